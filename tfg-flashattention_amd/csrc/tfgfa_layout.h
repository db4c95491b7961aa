// tfgfa_layout.h - the operand layouts that the serving operators take.
#ifndef TFGFA_LAYOUT_H
#define TFGFA_LAYOUT_H

#include <stdint.h>

#include <algorithm>
#include <utility>

namespace tfgfa {

struct Pages {  // byte strides of a (P, H_kv, page, D) cache of 16-bit elements
  long long p, h, n;
};
struct Rows {  // element strides of a (B, H, N, D) operand
  long long b, h, n;
};
struct Vecs {  // element strides of a (B, H, D) operand
  long long b, h;
};

// Last dimension dense, the others non-negative multiples of 8 elements, rows apart.  The stride of a dimension of
// one element (or none) is taken as 0.
inline bool rows_ok(const int64_t* st, long long B, long long H, long long N, int D, Rows* out) {
  const Rows r = {B <= 1 ? 0 : st[0], H <= 1 ? 0 : st[1], N <= 1 ? D : st[2]};
  if (st[3] != 1 || r.b < 0 || r.h < 0 || r.n < D || ((r.b | r.h | r.n) & 7)) return false;
  *out = r;
  return true;
}
inline bool pages_ok(const int64_t* st, int P, int H_kv, int page, int D, Pages* out) {
  Rows r;
  if (!rows_ok(st, P, H_kv, page, D, &r)) return false;
  *out = {2 * r.b, 2 * r.h, 2 * r.n};
  return true;
}
inline bool vecs_ok(const int64_t* st, long long B, long long H, Vecs* out) {
  const Vecs v = {B <= 1 ? 0 : st[0], H <= 1 ? 0 : st[1]};
  if (st[2] != 1 || v.b < 0 || v.h < 0 || ((v.b | v.h) & 7)) return false;
  *out = v;
  return true;
}

// Rows of `width` elements, na by nb of them at strides sa and sb, share none: the smaller stride is past the width,
// the larger past the span of the smaller.  A dimension of one has no stride.
inline bool apart(long long sa, long long na, long long sb, long long nb, long long width) {
  if (na <= 1 || (nb > 1 && sb < sa)) {
    std::swap(sa, sb);
    std::swap(na, nb);
  }
  long long reach = width - 1;
  if (na > 1) {
    if (sa <= reach) return false;
    reach += (na - 1) * sa;
  }
  return nb <= 1 || sb > reach;
}

// The rows of a pool (one that is written to) share none: of its strides from the smallest on, each is past the span of
// those before it.
inline bool pages_apart(const Pages& st, int P, int H_kv, int page, int D) {
  std::pair<long long, long long> dims[3] = {{st.p, P}, {st.h, H_kv}, {st.n, page}};
  std::sort(dims, dims + 3);
  __int128 reach = 2 * D - 1;
  for (const auto& d : dims) {
    if (d.second <= 1) continue;
    if (d.first <= reach) return false;
    reach += (__int128)(d.second - 1) * d.first;
  }
  return true;
}

// j / page = j * m >> s for 0 <= j < 2^31: with 2^(l-1) < page <= 2^l and m = floor(2^(31+l) / page) + 1 the error j (m
// page - 2^(31+l)) / (page 2^(31+l)) is below 1 / page, and m < 2^32.
struct Division {
  uint32_t m;
  int s;
};
inline Division division_by(int page) {
  int l = 0;
  while ((1LL << l) < page) ++l;
  return {(uint32_t)((1ULL << (31 + l)) / (uint64_t)page + 1), 31 + l};
}

}  // namespace tfgfa

#endif  // TFGFA_LAYOUT_H
