// tfgfa_weights.hip - the attention weight that each key receives from given queries, MI355X (gfx950):
//     c_j = sum_h sum_i [j <= first + i] e^(scale q_hi . k_j - lse_hi)
// over the query heads h of a key-value head, with the log-sum-exp of the attention that ran before.
//
// e^(x - lse) is 2^(c s - z) in one v_fma, c the scale times log2 e and z = lse log2 e, both rounded: off by 2^-24 (|c
// s| + |z|), as x - lse in float32 is.  Where a tile's |z| pass kCoarse, 64, what their roundings left is added (lse
// near 786432: sums 7% off without; a factor for it in every tile took 16 heads of 8192 from 101 to 112 us).
//
// Bound: VALU issue.  A pair of query and key costs 2D flops on the matrix units (128 cycles a 32x32 tile at D = 64)
// and a v_fma, a v_exp_f32 and a v_add on the VALU (16 x 15 cycles a tile).
// Measured: 16 heads of 8192 causal queries and keys, D = 64, 101-106 us (on different cards), 650-680 TFLOP/s; VALU
// issue 66% of the cycles, matrix units 25%, 38% of the wave cycles waiting to issue (without the exponentials 90 us,
// without the matrix products 73.5, without LDS reads 83, where the whole took 101).  D = 128, 4 x 16 heads of 4096:
// 163 us, 845 TFLOP/s.  64 queries against 16001 keys, 2 x 32 heads on 8, D = 128, 36 us, 28 where K is in the
// Infinity Cache, 12 of them a plain read of K: a workgroup's first loads are not covered.
//
// S^T[key][query] = K Q^T as v_mfma_f32_32x32x16 tiles: lane l holds 16 keys of query l % 32, so that the query's lse
// is one register, the sums over queries stay in 16 registers of each lane, and lanes are added once at the end.  A
// wave owns 32 keys of one key-value head, whose K rows stay in registers; the four waves of a workgroup share tiles
// of 64 queries, which come through two LDS buffers by direct loads, the next tile's under this one's arithmetic (an
// operand read straight from memory touches 32 rows an instruction, 32 bytes of each). Under a causal mask the first
// keys are seen by most queries.  Their workgroups come first; where several share a CU, every other round of
// workgroups over the CUs runs backwards, so that a CU's long and short ones add up alike (16 heads of 8192 queries
// and keys: 1024 workgroups, all resident, of which one CU had 160 parts and another 100; 100 us, in plain order
// 106).
// Tried and slower: 8 waves a workgroup (114 us), two key tiles a wave (139), the causal ends paired in one wave
// (163); for few queries, all of them in LDS and waves that go through the keys (27 -> 19 us for 32 queries, but 8.3
// -> 10.5 and 13.4 -> 15 at other sizes).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tfgfa.h"
#include "tfgfa_arrive.h"
#include "tfgfa_device.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_weights {

using tfgfa::apart;
using tfgfa::Rows;
using tfgfa::rows_ok;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLog2eHi = (float)kLog2e, kLog2eLo = (float)(kLog2e - kLog2eHi);
constexpr float kCoarse = 64.f;  // the largest |z| whose rounding is left at that
constexpr int kMaxD = 128;
constexpr int kTile = 32;              // keys of a wave, queries of a matrix tile
constexpr int kWaves = 4;
constexpr int kKeys = kTile * kWaves;  // keys of a workgroup
constexpr int kQueries = 64;           // queries of an LDS buffer
constexpr int kOutOfRange = 0x7FFFFFF0;  // a buffer offset past any num_records: the load gives zeros

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
  float scale_log2, scale_log2_rest;  // c, and what its rounding left
  int Hkv, units, cu, G, Nq, Nk, D, causal;
  // Where the queries of a block of keys are divided: parts, tiles of a part, arrival words and sums of parts.
  int splits, part_tiles;
  char* arrive;
  float* part;
  u64 tag;
};

// Rows of queries in LDS: kChunks chunks of 16 bytes, chunk c of row r at place c ^ turn(r), so that the rows of a
// chunk that a read takes together lie in different banks.
template <int kChunks>
__device__ __forceinline__ int turn(int row) {
  return kChunks == 8 ? tfgfa::swz_k(row) : row & 15;
}

// The sums over the 32 queries (lanes) of each half of the registers of s, 16 of them: halves of the registers change
// sides with the lanes that differ in one bit of their number (of the last ones three: any pairing does that flips
// the bit), so that each step adds half as many.  Lane l ends with register l / 2 % 16.
__device__ __forceinline__ float over_queries(const float (&sum)[16], int lane) {
  float s[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const auto two = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[r]), __float_as_uint(sum[r + 8]), false, false);
    s[r] = __uint_as_float(two[0]) + __uint_as_float(two[1]);
  }
  auto halve = [&](auto n, auto turned, int bit) {
#pragma unroll
    for (int r = 0; r < decltype(n)::value; ++r) {
      const float mine = lane & bit ? s[r + decltype(n)::value] : s[r], other = lane & bit ? s[r] : s[r + decltype(n)::value];
      s[r] = mine + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(other), decltype(turned)::value, 0xF, 0xF,
                                                               false));
    }
  };
  halve(std::integral_constant<int, 4>(), std::integral_constant<int, 0x128>(), 8);  // 8 lanes on
  halve(std::integral_constant<int, 2>(), std::integral_constant<int, 0x141>(), 4);  // mirrored in 8 lanes
  halve(std::integral_constant<int, 1>(), std::integral_constant<int, 0x4E>(), 2);   // 2 lanes on in 4
  return s[0] + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(s[0]), 0xB1, 0xF, 0xF, false));
}
// The key of a wave's 32 whose sum the lane ends with: register r of half h is key 8 (r / 4) + 4 h + r % 4.
__device__ __forceinline__ int key_of(int lane) {
  const int r = lane / 2 % 16;
  return 8 * (r / 4) + 4 * (lane / 32) + r % 4;
}

// kP: pieces of 16 dims, D <= 16 kP; a lane holds dims 16p + 8 (l / 32) .. + 7 of row l % 32.
// kSplit: a block of keys is several workgroups', each with part_tiles tiles of its queries; they leave their sums in the
// workspace, and the one that arrives last adds them in order (arrival words and memory order as in tfgfa_decode.hip).
template <class T, int kP, bool kSplit>
__global__ __launch_bounds__(64 * kWaves, 2) void weights_kernel(const Args a) {
  constexpr int kChunks = 2 * kP, kRowBytes = 16 * kChunks, kBytes = kQueries * kRowBytes;
  constexpr int kMoves = kBytes / 1024 / kWaves;  // 1-KiB transfers of a wave
  __shared__ __attribute__((aligned(1024))) unsigned char buf[2][kBytes];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, i = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x, piece = 0;
  if constexpr (kSplit) {
    id = blockIdx.x / a.splits;
    piece = blockIdx.x - id * a.splits;
  } else if (a.causal && id / a.cu % 2 != 0) {
    const int first = id / a.cu * a.cu;
    id = first + min(first + a.cu, (int)gridDim.x) - 1 - id;
  }
  const int y = id / a.units, unit = id - y * a.units;
  const int b = unit / a.Hkv, kv = unit - b * a.Hkv;
  const int jw = y * kKeys, j0 = jw + wave * kTile;  // first key of the workgroup, of the wave
  // Tiles of queries that see a key of this workgroup, for each of the head's query heads in turn.
  const int tiles = (a.Nq + kQueries - 1) / kQueries;
  int t0 = 0;
  if (a.causal && jw > a.first) t0 = (int)min((long long)tiles, (jw - a.first) / kQueries);
  const int per = tiles - t0;
  int all = per * a.G, parts = 1, from_tile = 0;
  u64* const aw = reinterpret_cast<u64*>(a.arrive + (long long)id * tfgfa::kArriveStride);
  u64 aw_start = 0;
  if constexpr (kSplit) {
    parts = max(1, (all + a.part_tiles - 1) / a.part_tiles);
    if (piece >= parts) return;
    from_tile = piece * a.part_tiles;
    all = min(a.part_tiles, all - from_tile);
    if (parts > 1 && tid == 0) aw_start = __hip_atomic_load(aw, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  u32x4 kf[kP];
  const T* const kr = static_cast<const T*>(a.k) + b * a.ks.b + kv * a.ks.h + (long long)(j0 + i) * a.ks.n + 8 * half;
#pragma unroll
  for (int p = 0; p < kP; ++p)
    kf[p] = j0 + i < a.Nk && 16 * p + 8 * half < a.D ? *reinterpret_cast<const u32x4*>(kr + 16 * p)
                                                     : u32x4{0, 0, 0, 0};

  const uint32_t at = tfgfa::lds_addr(&buf[0][0]);
  const int row_bytes = (int)a.qs.n * 2;
  // lse of the lane's query of each half of a tile, past the last query 0, and in the log2 domain; the next tile's.
  float lse_i[2], z[2], next[2];
  // The next tile's queries and their lse, and how many there are from it on in this head.
  int t = t0, h = kv * a.G;
  if (kSplit && per > 0) {
    const int g = __builtin_amdgcn_readfirstlane(from_tile / per);
    h += g, t += from_tile - g * per;
  }
  const T* q = static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h + (long long)t * kQueries * a.qs.n;
  const float* lse = a.lse + b * a.lb + h * a.lh + t * kQueries;
  const int left0 = a.Nq - t0 * kQueries;
  const long long q_tile = kQueries * a.qs.n;
  const long long q_head = a.qs.h - (long long)per * q_tile, lse_head = a.lh - (long long)per * kQueries;
  int left = a.Nq - t * kQueries;
  // The next tile into buffer n: lane l of a transfer writes 16 bytes at 16 l of its KiB.
  auto load = [&](int n) {
    const int rows = min(kQueries, left);
    const __amdgpu_buffer_rsrc_t z = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(lse), (short)0, rows * 4,
                                                                       0x00020000);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      next[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(z, (u * kTile + i) * 4, 0, 0));
    const tfgfa::i32x4 desc = tfgfa::head_desc(q, rows, row_bytes);
#pragma unroll
    for (int m = 0; m < kMoves; ++m) {
      const int first = (wave * kMoves + m) * (64 / kChunks), row = first + lane / kChunks;
      const int chunk = (lane & (kChunks - 1)) ^ turn<kChunks>(row);
      tfgfa::lds_transfer(desc, __builtin_amdgcn_readfirstlane(at + n * kBytes + first * kRowBytes),
                          8 * chunk < a.D ? row * row_bytes + 16 * chunk : kOutOfRange);
    }
    q += q_tile, lse += kQueries, left -= kQueries;
    if (left <= 0) q += q_head, lse += lse_head, left = left0;
  };

  float sum[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) sum[r] = 0.f;
  // The scale as a vector register: a v_fma with a scalar operand takes half as long again.
  float scale = a.scale_log2;
  asm("" : "+v"(scale));
  // Tiles from `from` to `upto` are seen whole by the wave's keys.
  int from = 0;
  if (a.causal && j0 + kTile - 1 > a.first)
    from = (int)min((long long)tiles, (j0 + kTile - 1 - a.first + kQueries - 1) / kQueries);
  const int upto = a.Nq / kQueries;
  if (all > 0) load(0);
#pragma unroll 1
  for (int w = 0; w < all; ++w) {
    const int n = w & 1;
    tfgfa::wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) lse_i[u] = next[u], z[u] = next[u] * kLog2eHi;
    if (w + 1 < all) load(n ^ 1);
    // Register r: key 8 (r / 4) + 4 half + r % 4 of the wave's, query i.
    auto scores = [&](int u) {
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
      const unsigned char* const row = &buf[n][(u * kTile + i) * kRowBytes];
#pragma unroll
      for (int p = 0; p < kP; ++p)
        s = mfma<T>(kf[p], *reinterpret_cast<const u32x4*>(row + 16 * ((2 * p + half) ^ turn<kChunks>(u * kTile + i))), s);
      return s;
    };
    const bool coarse = __builtin_amdgcn_ballot_w64(fmaxf(fabsf(z[0]), fabsf(z[1])) > kCoarse) != 0;
    if (t >= from && t < upto && !coarse) {
      const f32x16 s[2] = {scores(0), scores(1)};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r] += __builtin_amdgcn_exp2f(fmaf(s[u][r], scale, -z[u]));
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // Half a tile without a query, or whose last one sees none of the wave's keys.
        const int q0 = t * kQueries + u * kTile;
        if (q0 >= a.Nq || (a.causal && a.first + q0 + kTile - 1 < j0)) continue;
        const f32x16 s = scores(u);
        // Keys that the lane's query sees: up to `last`.  A row past the last, and one with nothing to see (lse -inf,
        // or past the range in the log2 domain), sees none.
        const bool live = fabsf(z[u]) != INFINITY && q0 + i < a.Nq;
        int last = kTile - 1;
        if (a.causal) last = (int)max(-1LL, min((long long)last, a.first + q0 + i - j0));
        if (!live) last = -1;
        const float zu = live ? z[u] : 0.f;
        auto add = [&](auto exponent) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            sum[r] += 8 * (r / 4) + 4 * half + r % 4 <= last ? __builtin_amdgcn_exp2f(exponent(s[r])) : 0.f;
        };
        if (coarse) {
          const float rest = live ? fmaf(lse_i[u], kLog2eLo, fmaf(lse_i[u], kLog2eHi, -z[u])) : 0.f;
          add([&](float x) { return fmaf(x, scale, -zu) + fmaf(x, a.scale_log2_rest, -rest); });
        } else {
          add([&](float x) { return fmaf(x, scale, -zu); });
        }
      }
    }
    if (++t == tiles) t = t0;
  }
  const int j = j0 + key_of(lane);
  const float x = over_queries(sum, lane);
  float* const out = a.out + b * a.ob + kv * a.oh;
  if (!kSplit || parts == 1) {
    if ((lane & 1) == 0 && j < a.Nk) out[j] = x;
    return;
  }
  if constexpr (kSplit) {
    __shared__ int sh_last;
    float* const mine = a.part + (long long)id * a.splits * kKeys;
    if ((lane & 1) == 0)
      __hip_atomic_store(mine + piece * kKeys + (j - jw), x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The part is at the coherence point once its stores are acknowledged; then the arrival is counted.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      if ((aw_start >> tfgfa::kTagShift) != a.tag) {
        u64 expected = aw_start;
        __hip_atomic_compare_exchange_strong(aw, &expected, a.tag << tfgfa::kTagShift, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT);
      }
      const u64 old = __hip_atomic_fetch_add(aw, (u64)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int last = (old & ((1ull << tfgfa::kTagShift) - 1)) == (u64)(parts - 1);
      if (last) __hip_atomic_store(aw, (u64)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh_last = last;
    }
    __syncthreads();
    if (!sh_last || tid >= kKeys || jw + tid >= a.Nk) return;
    asm volatile("" ::: "memory");
    float total = 0.f;
    constexpr int kBatch = 8;
    for (int s0 = 0; s0 < parts; s0 += kBatch) {
      float z[kBatch];
#pragma unroll
      for (int s = 0; s < kBatch; ++s)
        z[s] = s0 + s < parts
                   ? __hip_atomic_load(mine + (s0 + s) * kKeys + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                   : 0.f;
#pragma unroll
      for (int s = 0; s < kBatch; ++s) total += z[s];
    }
    out[jw + tid] = total;
  }
}

// ---------------------------------------------------------------------------------------
// Host side.

constexpr int kMaxCu = 1024;    // for the workspace's size, which does not depend on the device
// The least tiles of a part (16 heads on 1, 727 queries and keys, 3 sequences: 12.3 us, with 2 12.8, with 8 15.0; 512
// queries of 12 heads 7.6, 6.4, 8.7; 1369 of 16, D = 128, 15.7, 18.5, 16.3).
constexpr int kMinTiles = 4;
// The same where every CU has a block of keys already (16 heads of 2300 queries and keys: 20.0 us, not divided 26.1, with 4
// 26.5; 2 x 12 heads of 1500 15.4, 19.0, 17.7; 13 queries of 32 heads on 4 against 4415 keys, 3 sequences, not
// divided 13.5, with 4 17.4).
constexpr int kManyTiles = 8;
constexpr int kMaxSplits = 64;
// Workgroups of a CU that a division aims at (32 heads on 4, D = 80, 2081 queries: 36 us, with 2 49, with 8 38; 32 on 8, D
// = 128, 2 x 1504: 39.7, 38.7 and 45.9).
constexpr int kSlots = 4;

// Parts of a block of keys and tiles of a part on a device of `cu` CUs: 1 and 0 where the blocks of keys fill it, or have
// few queries.  (16 heads on 1, 2930 queries and keys: 26.5 us, not divided 482; 32 on 4, 1792: 23 and 145; 12 heads of
// 1024: 9.7 and 13.2.  Twice as many blocks as CUs divided too: 200 heads of 512, 13.4 -> 19.0.)
struct Split {
  int splits, tiles;
};
static Split choose_split(long long units, int G, int N_q, int N_k, int causal, int cu) {
  const long long blocks = (N_k + kKeys - 1) / kKeys * units, tiles = (long long)((N_q + kQueries - 1) / kQueries) * G;
  const int least = blocks < cu ? kMinTiles : kManyTiles;
  if (blocks >= 2LL * cu || tiles < 2 * least) return {1, 0};
  // (Under a causal mask about half the tiles are seen.)
  const long long share = blocks * tiles / (causal ? 2 : 1) / ((long long)kSlots * cu);
  const long long part = std::max<long long>({least, share, (tiles + kMaxSplits - 1) / kMaxSplits});
  return {(int)((tiles + part - 1) / part), (int)part};
}
// Blocks of keys, and tiles of queries of a key-value head, are counted in 32 bits.
static bool too_large(long long units, int G, int N_q, int N_k) {
  return units > INT32_MAX / 4096 || N_k > INT32_MAX - kKeys || (N_k / kKeys + 1) * units > INT32_MAX ||
         N_q > INT32_MAX - kQueries || (long long)(N_q / kQueries + 1) * G > INT32_MAX;
}
static size_t split_bytes(long long blocks, int splits) {
  return splits > 1 ? tfgfa::arrive_bytes(blocks) + (size_t)blocks * splits * kKeys * 4 : 0;
}

}  // namespace tfgfa_weights

extern "C" size_t tfserve_key_weights_workspace(int B, int H, int H_kv, int N_q, int N_k, int causal) {
  using namespace tfgfa_weights;
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || N_q <= 0 || N_k <= 0) return 0;
  const long long units = (long long)B * H_kv;
  if (too_large(units, H / H_kv, N_q, N_k)) return 0;
  // (A device of fewer CUs divides less.)
  const Split s = choose_split(units, H / H_kv, N_q, N_k, causal, kMaxCu);
  return split_bytes((long long)((N_k + kKeys - 1) / kKeys) * units, s.splits);
}

extern "C" int tfserve_key_weights(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const float* lse, const int64_t* lse_strides, float* out,
                                   const int64_t* out_strides, int B, int H, int H_kv, int N_q, int N_k, int D,
                                   int dtype, float softmax_scale, int causal, int64_t first_query,
                                   void* workspace, size_t workspace_bytes, void* hip_stream) {
  using namespace tfgfa_weights;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (B < 0 || H < 0 || H_kv < 0 || N_q < 0 || N_k < 0 || first_query < 0) return TFGFA_ERR_BAD_SHAPE;
  if (H_kv == 0 ? H != 0 : (H == 0 || H % H_kv != 0)) return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (!(softmax_scale > 0.f) || !isfinite(softmax_scale)) return TFGFA_ERR_SCALE;
  if (causal != 0 && causal != 1) return TFGFA_ERR_CAUSAL_FLAG;
  if (B == 0 || H == 0 || N_k == 0) return TFGFA_OK;
  const long long units = (long long)B * H_kv;
  if (too_large(units, H / H_kv, N_q, N_k) || first_query > INT64_MAX / 2) return TFGFA_ERR_TOO_LARGE;
  if (!q_strides || !k_strides || !lse_strides || !out_strides) return TFGFA_ERR_NULL_POINTER;
  Args a = {};
  if (!rows_ok(q_strides, B, H, N_q, D, &a.qs) || !rows_ok(k_strides, B, H_kv, N_k, D, &a.ks))
    return TFGFA_ERR_STRIDE;
  // A tile's rows are one buffer of less than 2^31 bytes.
  if (a.qs.n > INT32_MAX / (4 * kQueries)) return TFGFA_ERR_TOO_LARGE;
  if (!k || !out || (N_q > 0 && (!q || !lse))) return TFGFA_ERR_NULL_POINTER;
  if (((uintptr_t)q | (uintptr_t)k) & 15u) return TFGFA_ERR_ALIGNMENT;
  if ((((uintptr_t)lse | (uintptr_t)out) & 3u) || ((uintptr_t)workspace & 15u)) return TFGFA_ERR_ALIGNMENT;
  a.lb = B > 1 ? lse_strides[0] : 0, a.lh = H > 1 ? lse_strides[1] : 0;
  a.ob = B > 1 ? out_strides[0] : 0, a.oh = H_kv > 1 ? out_strides[1] : 0;
  if (a.lb < 0 || a.lh < 0 || !apart(a.ob, B, a.oh, H_kv, N_k))
    return TFGFA_ERR_STRIDE;
  a.q = q, a.k = k, a.lse = lse, a.out = out;
  a.first = first_query;
  a.scale_log2 = (float)(softmax_scale * kLog2e), a.scale_log2_rest = (float)(softmax_scale * kLog2e - a.scale_log2);
  a.Hkv = H_kv, a.G = H / H_kv, a.Nq = N_q, a.Nk = N_k, a.D = D, a.causal = causal;
  a.units = B * H_kv;
  const int st = tfgfa_device_info(&a.cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  const hipStream_t stream = (hipStream_t)hip_stream;
  const long long blocks = (long long)((N_k + kKeys - 1) / kKeys) * units;
  Split s = choose_split(units, a.G, N_q, N_k, causal, std::min(a.cu, kMaxCu));
  // Without a workspace that holds the parts, a block of keys is one workgroup's.
  if (split_bytes(blocks, s.splits) > (workspace ? workspace_bytes : 0)) s = {1, 0};
  a.splits = s.splits, a.part_tiles = s.tiles;
  a.arrive = static_cast<char*>(workspace);
  if (s.splits > 1) {
    a.part = reinterpret_cast<float*>(a.arrive + tfgfa::arrive_bytes(blocks));
    a.tag = tfgfa::next_tag();
  }
  const dim3 grid((unsigned)(blocks * s.splits));
#define TFGFA_WEIGHTS_(T, kP, kSplit) \
  hipLaunchKernelGGL((weights_kernel<T, kP, kSplit>), grid, dim3(64 * kWaves), 0, stream, a)
#define TFGFA_WEIGHTS(T)                                       \
  do {                                                         \
    if (D <= 64 && s.splits > 1) TFGFA_WEIGHTS_(T, 4, true);   \
    else if (D <= 64) TFGFA_WEIGHTS_(T, 4, false);             \
    else if (s.splits > 1) TFGFA_WEIGHTS_(T, 8, true);         \
    else TFGFA_WEIGHTS_(T, 8, false);                          \
  } while (0)
  if (dtype == TFGFA_DTYPE_BF16)
    TFGFA_WEIGHTS(__bf16);
  else
    TFGFA_WEIGHTS(_Float16);
#undef TFGFA_WEIGHTS
#undef TFGFA_WEIGHTS_
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
