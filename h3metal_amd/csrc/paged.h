// What the kernels over a paged cache share. A cache holds keys and values as [pages][heads][page][channels] of 16-bit
// elements each; row c of sequence b is row c % page of page table[b][c / page]. A batch's new tokens are consecutive rows,
// those of sequence b from q_start[b] to q_start[b + 1] - 1, and its last one is the sequence's last row, kv_len[b] - 1. All
// three live in device memory (a call reads what they hold when it runs), so the host cannot check them: the kernels do, and
// whatever they hold, no access leaves its buffer.
#pragma once

#include "h3hip_internal.h"

#include <string>

namespace h3 {

// Where the batch's rows are.
struct Batch {
  const int *table, *q_start, *kv_len;
  int B, width, pages, lg;  // sequences, pages a row of the table names, pages of the cache, log2 of a page's rows
};

namespace {

enum { P_BF16 = 0, P_F16 = 1, P_F32 = 2 };
template <int T> struct PElem;
template <> struct PElem<P_BF16> { using type = __bf16; };
template <> struct PElem<P_F16> { using type = _Float16; };
template <> struct PElem<P_F32> { using type = float; };

// Host side: the checks both operators make of an argument and of the page table's shape.
inline bool paged_fits(const Arg *a, int i, uint64_t bytes, int align, const char *what, std::string *err) {
  if (!a[i].ptr) {
    *err = std::string(what) + " is not bound";
    return false;
  }
  if (bytes > a[i].avail) {
    *err = std::string(what) + " needs " + std::to_string(bytes) + " bytes, its buffer holds " + std::to_string(a[i].avail);
    return false;
  }
  if ((uintptr_t)a[i].ptr % align) {
    *err = std::string(what) + " must be " + std::to_string(align) + "-byte aligned";
    return false;
  }
  return true;
}
inline bool paged_overlap(const Arg &p, uint64_t n, const Arg &q, uint64_t k) {
  return n && k && p.ptr && q.ptr && p.ptr < q.ptr + k && q.ptr < p.ptr + n;
}
inline int log2_page(int page) {  // -1: not a power of two from 16 to 256
  for (int lg = 4; lg <= 8; lg++)
    if (page == 1 << lg) return lg;
  return -1;
}
inline int paged_type(const std::string &s) {
  return s == "bfloat" || s == "bf16" ? P_BF16 : s == "half" || s == "f16" ? P_F16 : s == "float" || s == "f32" ? P_F32 : -1;
}

}  // namespace
}  // namespace h3
