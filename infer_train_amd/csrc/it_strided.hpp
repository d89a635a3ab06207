// it_strided.hpp -- whether two sets of rows in memory share a byte (host).
#pragma once
#include <cstdint>

namespace itkv {

// n_tokens x n_heads rows of `bytes` bytes each, `token` and `head` bytes apart (0 and more).
struct StridedRows {
  uintptr_t at;
  int64_t token, head, bytes;
  int64_t n_tokens, n_heads;
  int64_t span() const { return (n_tokens - 1) * token + (n_heads - 1) * head + bytes; }
};

// Exact where the rows of both are equally many tokens apart (parts of one
// projection: rows of one may lie between those of the other), or of one token;
// else rows that lie between one another count as shared.
inline bool share_memory(const StridedRows& a, const StridedRows& b) {
  if (a.n_tokens <= 0 || b.n_tokens <= 0 || a.n_heads <= 0 || b.n_heads <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
  if (a.at >= b.at + uintptr_t(b.span()) || b.at >= a.at + uintptr_t(a.span())) return false;
  if ((a.n_tokens > 1 || b.n_tokens > 1) && (a.token != b.token || a.n_tokens != b.n_tokens || a.token <= 0)) return true;
  const int64_t base = int64_t(b.at) - int64_t(a.at), far = a.n_tokens - 1;
  // Whether rows of a and b whose heads are `apart` bytes from one another meet in any two tokens: a's
  // begin at 0, b's at x = apart + d * token for d from -far to far, and -b.bytes < x < a.bytes.  The
  // least d for the left side is tried against the right one.
  const auto meet = [&](int64_t apart) {
    if (far == 0) return apart > -b.bytes && apart < a.bytes;
    const int64_t over = -b.bytes - apart;
    int64_t d = over / a.token + (over % a.token != 0 && over < 0 ? 0 : 1);  // floor(over / token) + 1
    if (d < -far) d = -far;
    return d <= far && apart + d * a.token < a.bytes;
  };
  if (a.head == b.head || a.n_heads == 1 || b.n_heads == 1) {  // what matters is the difference of their heads' numbers
    const int64_t head = a.n_heads > 1 ? a.head : b.head;
    for (int64_t d = 1 - a.n_heads; d < b.n_heads; ++d)
      if (meet(base + d * head)) return true;
    return false;
  }
  if (a.n_heads * b.n_heads > int64_t(1) << 16) return true;
  for (int64_t i = 0; i < a.n_heads; ++i)
    for (int64_t j = 0; j < b.n_heads; ++j)
      if (meet(base + j * b.head - i * a.head)) return true;
  return false;
}

}  // namespace itkv
