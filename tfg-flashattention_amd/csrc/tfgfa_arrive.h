// tfgfa_arrive.h - the arrival words of workgroups that divide one piece of work and have the last
// of them join the parts (protocol: tfgfa_decode.hip).
#ifndef TFGFA_ARRIVE_H
#define TFGFA_ARRIVE_H

#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <chrono>

namespace tfgfa {

constexpr int kArriveStride = 128;  // bytes between the arrival words of two pieces of work
constexpr int kTagShift = 16;       // arrival word: tag << 16 | count (count < 2^16)

// Bytes of the arrival words at the start of a workspace: one per piece, kArriveStride apart.
inline size_t arrive_bytes(long long pieces) {
  return ((size_t)pieces * kArriveStride + 255) / 256 * 256;
}

// A random nonzero 48-bit tag per call (splitmix64 over a process-wide counter and a seed from
// the clock and an address), so that no word left in memory by anything else is likely to
// carry it.
inline uint64_t splitmix64(uint64_t x) {
  x += 0x9E3779B97F4A7C15ull;
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}
inline uint64_t next_tag() {
  static std::atomic<uint64_t> counter{0};
  static const uint64_t seed =
      splitmix64((uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() ^
                 (uint64_t)(uintptr_t)&counter);
  const uint64_t t = splitmix64(seed + counter.fetch_add(1, std::memory_order_relaxed)) &
                     ((1ull << (64 - kTagShift)) - 1);
  return t ? t : 1;
}

}  // namespace tfgfa

#endif  // TFGFA_ARRIVE_H
