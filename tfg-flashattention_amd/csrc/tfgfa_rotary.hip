// tfgfa_rotary.hip - rotary positions, and new tokens' keys and values into a paged cache with the rotation on the
// way, MI355X (gfx950); float32, bf16 and fp16.
//
//     y_a = m (x_a cos t - x_b sin t),   y_b = m (x_b cos t + x_a sin t),   t = position f_i
// for the pairs (a, b) = (i, i + r/2) or (2i, 2i + 1) of the first r dims; the others are copied.  The transposed
// rotation (-t for t) is the gradient's.
//
// Angles.  f_i comes as turns of a position in 2^-64, a 64-bit integer: position * turns modulo 2^64 is the exact
// phase, at any position, and its upper 32 bits are the phase to 2^-33 of a turn (position * f_i in float32 is off by
// 0.03 radians at position 10^6).  Quarter turns are taken off as integers; what is left, |x| <= pi/4, is off by two
// roundings (2^-24 each, relative), and the Taylor series end below 2^-25 (x^11/11! for the sine, x^12/12! for the cosine).
//
// Bound: HBM, every element read and written once.  A workgroup takes some tokens with all their heads: sines and
// cosines of a token are computed once, into LDS, for all heads of queries and keys, as is where its rows lie (a
// row's page among it); then each thread moves the same 16 bytes of each token, or two times 16 of a pair of halves, so that
// heads and places in them are told apart once.  (Told apart for each piece, 57 and 100 us for the appends below.)
// Measured, from memory, us and TB/s read and written: 32001 tokens of 32 + 8 heads, half of each rotated, fp16, 132 (5.0;
// a copy of as many bytes 127); 16000 of them in float32 138 (4.8); 2 chunks of 8192 tokens into pages, queries too, 80 (5.0); 16 prompts of up to 1024 tokens,
// 25 heads, into pages 31.3 (3.8: 40% of the padded batch's tokens are looked at and left, and the 400 items of a token leave
// 22% of two rounds of threads idle); 8 tokens 3.2.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tfgfa.h"
#include "tfgfa_layout.h"
#include "tfgfa_pages.h"

namespace tfgfa_rotary {

using tfgfa::Pages;
using tfgfa::Rows;

constexpr int kThreads = 256;
constexpr int kMaxD = 128;
constexpr int kMaxTokens = 16;   // of a workgroup
constexpr int kMaxRun = 1 << 27;  // of a launch: workgroups of more than kMaxTokens / 2 then have fewer than 2^32 threads
constexpr int kTensors = 3;      // of a launch
constexpr int kItems = 2;        // tokens of a thread in flight

// One tensor of the launch.  Its heads' vectors are moved in items: `turned` of them rotate pairs, then `single` copy an
// element each from dim r on, and `wide` copy 16 bytes.
struct Tensor {
  const void* x;
  void* y;
  long long xb, xh, xn, yb, yh, yn;  // element strides; in pages: yb is a page's
  int heads, turned, single, wide;
  int first;                         // of a token's items
};

struct Args {
  Tensor t[kTensors];
  const uint64_t* turns;
  const void* positions;
  long long pb, pn, first;           // positions: element strides; first where there are none
  int position_bytes;                // 0: none
  float magnitude, sign;
  int rot, N, tokens;                // tokens: B * N
  int each, parts, count;            // tokens of a workgroup, workgroups that share them, tensors
  int items;                         // of a token
  int side, slots;                   // tokens that the workgroup's threads take side by side; rounds of threads for them
  tfgfa::Division by_items;
  // Pages (tensors 0 and 1, K and V; tensor 2 is Q).
  const int* table;
  const int* lens;
  const int* lengths;
  long long table_stride;
  tfgfa::Division by_page;
  int page, P, n_max, pad;
};

// What becomes of a token's rows.
enum Fate : int { kMove, kSkip, kZero, kNan };

__device__ __forceinline__ int divide(int x, tfgfa::Division d) { return (int)(((uint64_t)(uint32_t)x * d.m) >> d.s); }

// Sine and cosine of p 2^-32 turns.
__device__ __forceinline__ void sin_cos(uint32_t p, float* s, float* c) {
  const uint32_t j = (p + 0x20000000u) >> 30;
  const float x = (float)(int)(p - (j << 30)) * 0x1.921fb6p-30f;  // 2 pi 2^-32
  const float z = x * x;
  const float u = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float v = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float a = j & 1 ? v : u, b = j & 1 ? u : v;
  *s = j & 2 ? -a : a;
  *c = (j + 1) & 2 ? -b : b;
}

// kHalves: pairs (i, i + r/2), an item two times kWide neighbouring dims; kNeighbours: pairs (2i, 2i + 1), an item kWide
// dims; kAny: an item one pair, for sizes and layouts where neither is whole 16-byte pieces: rotated dims that are no
// multiple of 16 (halves) or 8 (neighbours) 16-bit elements, of 8 or 4 float32 ones, and unaligned views.  (32001 tokens of 32 + 8
// heads of 128, fp16: 20 dims rotated in halves 221 us, 40 234, 20 of neighbours 227, for 130 to 132 with 64 or 128; heads of
// 40 rotated whole 112, for the 41 of a copy; 16000 tokens in float32 175 with 20 dims, 138 with 64.)
enum class Pairs { kHalves, kNeighbours, kAny };

template <class E, Pairs kPairs, bool kPaged>
__global__ __launch_bounds__(kThreads) void rotate_kernel(const Args a, int interleaved) {
  constexpr int kWide = 16 / sizeof(E);
  typedef E wide __attribute__((ext_vector_type(kWide)));
  constexpr int kEach = kPairs == Pairs::kHalves ? kWide : kPairs == Pairs::kNeighbours ? kWide / 2 : 1;  // pairs of an item
  __shared__ __attribute__((aligned(16))) float sh_cos[kMaxTokens * kMaxD / 2], sh_sin[kMaxTokens * kMaxD / 2];
  __shared__ long long sh_x[kTensors][kMaxTokens], sh_y[kTensors][kMaxTokens];
  __shared__ int sh_fate[kTensors][kMaxTokens];
  const int tid = threadIdx.x, part = (int)(blockIdx.x % (unsigned)a.parts);
  const int u0 = (int)(blockIdx.x / (unsigned)a.parts) * a.each, here = min(a.each, a.tokens - u0);
  const int pairs = a.rot / 2;

  auto position = [&](int b, int n) -> long long {
    if constexpr (kPaged) return (long long)(a.position_bytes ? static_cast<const int*>(a.positions)[b] : a.lens[b]) + n;
    const long long at = b * a.pb + n * a.pn;
    return a.position_bytes == 8   ? static_cast<const long long*>(a.positions)[at]
           : a.position_bytes == 4 ? (long long)static_cast<const int*>(a.positions)[at]
                                   : a.first + n;
  };
  for (int e = tid; e < here * pairs; e += kThreads) {
    const int t = e / pairs, i = e - t * pairs, b = (u0 + t) / a.N, n = u0 + t - b * a.N;
    const uint64_t phase = (uint64_t)position(b, n) * a.turns[i];
    float s, c;
    sin_cos((uint32_t)((phase + 0x80000000u) >> 32), &s, &c);
    sh_cos[t * pairs + i] = c * a.magnitude;
    sh_sin[t * pairs + i] = s * a.magnitude * a.sign;
  }
  // The last threads, which have the fewest angles to compute, find the rows.
  if (kThreads - 1 - tid < here) {
    const int t = kThreads - 1 - tid, b = (u0 + t) / a.N, n = u0 + t - b * a.N;
#pragma unroll
    for (int s = 0; s < kTensors; ++s) {
      sh_x[s][t] = b * a.t[s].xb + n * a.t[s].xn;
      sh_y[s][t] = b * a.t[s].yb + n * a.t[s].yn;
      sh_fate[s][t] = kMove;
    }
    if constexpr (kPaged) {
      const int len = a.lens[b], count = a.lengths ? a.lengths[b] : a.N;
      const bool fits = len >= 0 && count >= 0 && count <= a.N && (long long)len + count <= a.n_max;
      int home = -1, row = 0;
      if (fits && n < count) {
        const int at = divide(len + n, a.by_page);
        home = a.table[b * a.table_stride + at];
        row = len + n - at * a.page;
      }
      const bool in = (uint32_t)home < (uint32_t)a.P;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        sh_y[s][t] = in ? home * a.t[s].yb + row * a.t[s].yn : 0;
        sh_fate[s][t] = in ? kMove : kSkip;
      }
      sh_fate[2][t] = !fits ? kNan : n < count ? kMove : a.pad ? kZero : kSkip;
    }
  }
  __syncthreads();

  // Each thread takes the same place of every `side`-th token: what tells the places apart is worked out once for them all.
  for (int slot = part; slot < a.slots; slot += a.parts) {
    const int place = slot * kThreads + tid, t0 = divide(place, a.by_items);
    if (t0 >= a.side) continue;
    int i = place - t0 * a.items;
    const int s = a.count > 2 && i >= a.t[2].first ? 2 : a.count > 1 && i >= a.t[1].first ? 1 : 0;
    // (Selected field by field: a pointer to one of the three would put the arguments in memory.)
    auto of = [&](auto f) { return s == 2 ? f(a.t[2]) : s == 1 ? f(a.t[1]) : f(a.t[0]); };
    i -= of([](const Tensor& z) { return z.first; });
    const int turned = of([](const Tensor& z) { return z.turned; }), single = of([](const Tensor& z) { return z.single; });
    const int per = turned + single + of([](const Tensor& z) { return z.wide; });
    const int h = (int)(((float)i + 0.5f) * __builtin_amdgcn_rcpf((float)per));  // exact: i < 2^21
    i -= h * per;
    const bool rotates = i < turned;
    int lo_at, hi_at = 0, angle = 0;
    bool one = false, two = false;  // an element instead of a piece; a second one
    if (rotates) {
      angle = i * kEach;
      if constexpr (kPairs == Pairs::kHalves) {
        lo_at = i * kWide, hi_at = lo_at + pairs, two = true;
      } else if constexpr (kPairs == Pairs::kNeighbours) {
        lo_at = i * kWide;
      } else {
        lo_at = interleaved ? 2 * i : i, hi_at = interleaved ? 2 * i + 1 : i + pairs, one = two = true;
      }
    } else {
      const int from = turned ? a.rot : 0;
      one = i < turned + single;
      lo_at = one ? from + i - turned : from + single + (i - turned - single) * kWide;
    }
    const E* const x = static_cast<const E*>(of([](const Tensor& z) { return z.x; })) + h * of([](const Tensor& z) { return z.xh; }) + lo_at;
    E* const y = static_cast<E*>(of([](const Tensor& z) { return z.y; })) + h * of([](const Tensor& z) { return z.yh; }) + lo_at;
    const int apart = hi_at - lo_at;
    for (int t = t0; t < here; t += a.side * kItems) {
      wide lo[kItems], hi[kItems];
      int fate[kItems];
#pragma unroll
      for (int m = 0; m < kItems; ++m) {
        const int u = t + m * a.side;
        fate[m] = u < here ? (kPaged ? sh_fate[s][u] : (int)kMove) : (int)kSkip;
        if (fate[m] != kMove) continue;
        const E* const from = x + sh_x[s][u];
        if (one)
          lo[m][0] = from[0];
        else
          lo[m] = *reinterpret_cast<const wide*>(from);
        if constexpr (kPairs == Pairs::kHalves) {
          if (two) hi[m] = *reinterpret_cast<const wide*>(from + apart);
        } else if constexpr (kPairs == Pairs::kAny) {
          if (two) hi[m][0] = from[apart];
        }
      }
#pragma unroll
      for (int m = 0; m < kItems; ++m) {
        const int u = t + m * a.side;
        if (fate[m] == kSkip) continue;
        if (fate[m] != kMove) {
          const E fill = (E)(fate[m] == kNan ? __uint_as_float(0x7FC00000u) : 0.f);
#pragma unroll
          for (int e = 0; e < kWide; ++e) lo[m][e] = fill, hi[m][e] = fill;
        } else if (rotates) {
          const float* const c = sh_cos + u * pairs + angle;
          const float* const sn = sh_sin + u * pairs + angle;
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const bool beside = kPairs == Pairs::kNeighbours;
            const float xa = (float)lo[m][beside ? 2 * e : e], xb = (float)(beside ? lo[m][2 * e + 1] : hi[m][e]);
            const E ya = (E)fmaf(xa, c[e], -(xb * sn[e])), yb = (E)fmaf(xb, c[e], xa * sn[e]);
            if (beside)
              lo[m][2 * e] = ya, lo[m][2 * e + 1] = yb;
            else
              lo[m][e] = ya, hi[m][e] = yb;
          }
        }
        E* const to = y + sh_y[s][u];
        if (one)
          to[0] = lo[m][0];
        else
          *reinterpret_cast<wide*>(to) = lo[m];
        if constexpr (kPairs == Pairs::kHalves) {
          if (two) *reinterpret_cast<wide*>(to + apart) = hi[m];
        } else if constexpr (kPairs == Pairs::kAny) {
          if (two) to[apart] = hi[m][0];
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side.

// A (B, H, N, D) operand whose last dimension is dense and whose other strides are not negative; those of dimensions of
// one element are taken as 0.
static bool takes_strides(const int64_t* st, long long B, long long H, long long N, int D, Rows* out) {
  const Rows r = {B <= 1 ? 0 : st[0], H <= 1 ? 0 : st[1], N <= 1 ? 0 : st[2]};
  if ((D > 1 && st[3] != 1) || r.b < 0 || r.h < 0 || r.n < 0) return false;
  *out = r;
  return true;
}

// Its vectors share no element.
static bool vectors_apart(const Rows& r, long long B, long long H, long long N, int D) {
  std::pair<long long, long long> dims[3] = {{r.b, B}, {r.h, H}, {r.n, N}};
  std::sort(dims, dims + 3);
  __int128 reach = D - 1;
  for (const auto& d : dims) {
    if (d.second <= 1) continue;
    if (d.first <= reach) return false;
    reach += (__int128)(d.second - 1) * d.first;
  }
  return true;
}

static bool same(const Rows& x, const Rows& y) { return x.b == y.b && x.h == y.h && x.n == y.n; }

// The tensor's items of a token.  pieces: 16-byte pieces are whole (its strides, and D); rot 0: it is copied.
static void set_items(Tensor* t, Pairs pairs, bool pieces, int wide, int rot, int D, bool copy_rest) {
  t->turned = pairs == Pairs::kHalves ? rot / 2 / wide : pairs == Pairs::kNeighbours ? rot / wide : rot / 2;
  t->single = t->wide = 0;
  if (!copy_rest) return;
  t->single = pieces ? std::min(D, (rot + wide - 1) / wide * wide) - rot : D - rot;
  t->wide = (D - rot - t->single) / wide;
}

// (a.t, count and tokens are set.)
template <class E, bool kPaged>
static int launch(Args a, Pairs pairs, int interleaved, int cu, hipStream_t stream) {
  long long items = 0;
  for (int s = 0; s < a.count; ++s) {
    a.t[s].first = (int)items;
    items += (long long)a.t[s].heads * (a.t[s].turned + a.t[s].single + a.t[s].wide);
    if (items >= 1 << 21) return TFGFA_ERR_TOO_LARGE;
  }
  if (items == 0) return TFGFA_OK;
  a.items = (int)items;
  a.by_items = tfgfa::division_by(a.items);
  a.side = (int)std::max(1LL, kThreads / items);
  a.slots = (int)((a.side * items + kThreads - 1) / kThreads);
  // As many tokens a workgroup as leave sixteen workgroups a CU; where there are fewer tokens, their places are divided.
  // (With 8 a CU 32001 tokens of 40 heads take 145 us, with 16 132, with 32 137, with 64 169; 16 prompts of up to 1024
  // tokens into pages 33.9, 31.3, 36.8, 55.)
  a.each = a.side;
  while (2 * a.each <= kMaxTokens && a.tokens / (2 * a.each) >= 16LL * cu) a.each *= 2;
  a.each = std::min(a.each, kMaxTokens);
  const long long groups = (a.tokens + a.each - 1) / a.each;
  a.parts = (int)std::max(1LL, std::min<long long>(a.slots, 4LL * cu / groups));
  const dim3 grid((unsigned)(groups * a.parts));
  if (pairs == Pairs::kHalves)
    hipLaunchKernelGGL((rotate_kernel<E, Pairs::kHalves, kPaged>), grid, dim3(kThreads), 0, stream, a, interleaved);
  else if (pairs == Pairs::kNeighbours)
    hipLaunchKernelGGL((rotate_kernel<E, Pairs::kNeighbours, kPaged>), grid, dim3(kThreads), 0, stream, a, interleaved);
  else
    hipLaunchKernelGGL((rotate_kernel<E, Pairs::kAny, kPaged>), grid, dim3(kThreads), 0, stream, a, interleaved);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}

static Pairs choose_pairs(bool pieces, int rot, int interleaved, int wide) {
  if (!pieces || rot % (interleaved ? wide : 2 * wide)) return Pairs::kAny;
  return interleaved ? Pairs::kNeighbours : Pairs::kHalves;
}

}  // namespace tfgfa_rotary

extern "C" int tfpages_rotate(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int H,
                              const void* k, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides,
                              int H_kv, const void* positions, int position_bytes, const int64_t* position_strides,
                              int64_t first, const uint64_t* turns, int rot, int interleaved, float magnitude,
                              int transposed, int B, int N, int D, int dtype, void* hip_stream) {
  using namespace tfgfa_rotary;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16 && dtype != TFPAGES_DTYPE_F32) return TFGFA_ERR_DTYPE;
  if (positions && position_bytes != 4 && position_bytes != 8) return TFGFA_ERR_DTYPE;
  if (B < 0 || H < 0 || H_kv < 0 || N < 0 || (unsigned)interleaved > 1 || (unsigned)transposed > 1) return TFGFA_ERR_BAD_SHAPE;
  if (D < 1 || D > kMaxD || rot < 0 || rot > D || (rot & 1)) return TFGFA_ERR_HEAD_DIM;
  if (!(magnitude > 0.f) || !isfinite(magnitude)) return TFGFA_ERR_SCALE;
  if (B == 0 || N == 0 || (H == 0 && H_kv == 0)) return TFGFA_OK;
  if ((long long)B * N > kMaxRun) return TFGFA_ERR_TOO_LARGE;
  if (rot > 0 && !turns) return TFGFA_ERR_NULL_POINTER;
  if (positions && !position_strides) return TFGFA_ERR_NULL_POINTER;
  const uintptr_t size = dtype == TFPAGES_DTYPE_F32 ? 4 : 2;
  const int wide = 16 / (int)size;
  Args a = {};
  bool pieces = D % wide == 0;
  const struct {
    const void* x;
    const int64_t* xs;
    void* y;
    const int64_t* ys;
    int heads;
  } given[2] = {{q, q_strides, q_out, q_out_strides, H}, {k, k_strides, k_out, k_out_strides, H_kv}};
  bool in_place[kTensors] = {};
  for (const auto& g : given) {
    if (g.heads == 0) continue;
    if (!g.x || !g.y || !g.xs || !g.ys) return TFGFA_ERR_NULL_POINTER;
    Rows x, y;
    if (!takes_strides(g.xs, B, g.heads, N, D, &x) || !takes_strides(g.ys, B, g.heads, N, D, &y)) return TFGFA_ERR_STRIDE;
    if (!vectors_apart(y, B, g.heads, N, D) || (g.x == g.y && !same(x, y))) return TFGFA_ERR_STRIDE;
    if (((uintptr_t)g.x | (uintptr_t)g.y) & (size - 1)) return TFGFA_ERR_ALIGNMENT;
    pieces = pieces && !(((uintptr_t)g.x | (uintptr_t)g.y) & 15u) && (x.b | x.h | x.n | y.b | y.h | y.n) % wide == 0;
    in_place[a.count] = g.x == g.y;
    a.t[a.count++] = {g.x, g.y, x.b, x.h, x.n, y.b, y.h, y.n, g.heads, 0, 0, 0, 0};
  }
  if (((uintptr_t)turns & 7u) || (positions && ((uintptr_t)positions & (position_bytes - 1)))) return TFGFA_ERR_ALIGNMENT;
  const Pairs pairs = choose_pairs(pieces, rot, interleaved, wide);
  for (int s = 0; s < a.count; ++s) set_items(&a.t[s], pairs, pieces, wide, rot, D, !in_place[s]);
  a.turns = turns, a.rot = rot, a.magnitude = magnitude, a.sign = transposed ? -1.f : 1.f;
  a.positions = positions, a.first = first, a.position_bytes = positions ? position_bytes : 0;
  if (positions) a.pb = position_strides[0], a.pn = position_strides[1];
  a.N = N, a.tokens = B * N;
  int cu = 0;
  const int st = tfgfa_device_info(&cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (dtype == TFGFA_DTYPE_BF16) return launch<__bf16, false>(a, pairs, interleaved, cu, stream);
  if (dtype == TFGFA_DTYPE_F16) return launch<_Float16, false>(a, pairs, interleaved, cu, stream);
  return launch<float, false>(a, pairs, interleaved, cu, stream);
}

extern "C" int tfpages_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                              void* k_pages, const int64_t* k_pages_strides, void* v_pages,
                              const int64_t* v_pages_strides, const int* page_table, int64_t table_stride,
                              const int* cache_seqlens, const int* lengths, const int* positions, const void* q,
                              const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int pad,
                              const uint64_t* turns, int rot, int interleaved, float magnitude, int B, int H,
                              int H_kv, int N, int P, int page, int M, int D, int dtype, void* hip_stream) {
  using namespace tfgfa_rotary;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (B < 0 || H < 0 || H_kv < 0 || N < 0 || P < 0 || page < 1 || M < 0 || (unsigned)interleaved > 1)
    return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7) || rot < 0 || rot > D || (rot & 1)) return TFGFA_ERR_HEAD_DIM;
  if (!(magnitude > 0.f) || !isfinite(magnitude)) return TFGFA_ERR_SCALE;
  if ((q == nullptr) != (q_out == nullptr)) return TFGFA_ERR_NULL_POINTER;
  if (H_kv == 0 && q && H > 0) return TFGFA_ERR_BAD_SHAPE;  // queries of a cache without heads
  if (B == 0 || N == 0 || H_kv == 0) return TFGFA_OK;
  const long long n_max = (long long)M * page;
  if ((long long)B * N > kMaxRun || n_max > INT32_MAX - kMaxTokens) return TFGFA_ERR_TOO_LARGE;
  if (!k || !v || !k_pages || !v_pages || !cache_seqlens || (!page_table && M > 0) || !k_strides || !v_strides ||
      !k_pages_strides || !v_pages_strides || (rot > 0 && !turns))
    return TFGFA_ERR_NULL_POINTER;
  Rows ks, vs;
  Pages kp, vp;
  if (!tfgfa::rows_ok(k_strides, B, H_kv, N, D, &ks) || !tfgfa::rows_ok(v_strides, B, H_kv, N, D, &vs) ||
      !tfgfa::pages_ok(k_pages_strides, P, H_kv, page, D, &kp) || !tfgfa::pages_ok(v_pages_strides, P, H_kv, page, D, &vp) ||
      !tfgfa::pages_apart(kp, P, H_kv, page, D) || !tfgfa::pages_apart(vp, P, H_kv, page, D))
    return TFGFA_ERR_STRIDE;
  if (B > 1 && table_stride < 0) return TFGFA_ERR_STRIDE;
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)q | (uintptr_t)q_out) & 15u)
    return TFGFA_ERR_ALIGNMENT;
  if ((((uintptr_t)page_table | (uintptr_t)cache_seqlens | (uintptr_t)lengths | (uintptr_t)positions) & 3u) ||
      ((uintptr_t)turns & 7u))
    return TFGFA_ERR_ALIGNMENT;
  Args a = {};
  a.t[0] = {k, k_pages, ks.b, ks.h, ks.n, kp.p / 2, kp.h / 2, kp.n / 2, H_kv, 0, 0, 0, 0};
  a.t[1] = {v, v_pages, vs.b, vs.h, vs.n, vp.p / 2, vp.h / 2, vp.n / 2, H_kv, 0, 0, 0, 0};
  a.count = 2;
  if (q && H > 0) {
    Rows qs, os;
    if (!q_strides || !q_out_strides) return TFGFA_ERR_NULL_POINTER;
    if (!tfgfa::rows_ok(q_strides, B, H, N, D, &qs) || !tfgfa::rows_ok(q_out_strides, B, H, N, D, &os) ||
        !vectors_apart(os, B, H, N, D) || (q == q_out && !same(qs, os)))
      return TFGFA_ERR_STRIDE;
    a.t[2] = {q, q_out, qs.b, qs.h, qs.n, os.b, os.h, os.n, H, 0, 0, 0, 0};
    a.count = 3;
  }
  constexpr int kWide = 8;
  const Pairs pairs = choose_pairs(true, rot, interleaved, kWide);
  for (int s = 0; s < a.count; ++s) set_items(&a.t[s], pairs, true, kWide, s == 1 ? 0 : rot, D, true);
  a.turns = turns, a.rot = rot, a.magnitude = magnitude, a.sign = 1.f;
  a.positions = positions, a.position_bytes = positions ? 4 : 0;
  a.N = N, a.tokens = B * N;
  a.table = page_table, a.table_stride = B > 1 ? table_stride : 0, a.lens = cache_seqlens, a.lengths = lengths;
  a.by_page = tfgfa::division_by(page), a.page = page, a.P = P, a.n_max = (int)n_max, a.pad = pad != 0;
  int cu = 0;
  const int st = tfgfa_device_info(&cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  const hipStream_t stream = (hipStream_t)hip_stream;
  return dtype == TFGFA_DTYPE_BF16 ? launch<__bf16, true>(a, pairs, interleaved, cu, stream)
                                   : launch<_Float16, true>(a, pairs, interleaved, cu, stream);
}
