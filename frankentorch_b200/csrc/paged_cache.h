// Where a position of a sequence is in a paged key-value cache.  Compiled by the kernels and, on its own, by a host test.
#pragma once

#ifdef __CUDACC__
#define FT_PAGED_FN __host__ __device__ __forceinline__
#else
#define FT_PAGED_FN inline
#endif

namespace ftk {

// The part of a page table that belongs to one cache: pages of 1 << shift rows, `cols` table entries per sequence.
struct PagedTable {
  const int* table;
  long long stride;
  long long cols;
  long long n_pages;
  int shift;
};

// Page of `position` of sequence `b`, or -1 where the table has no entry for it or the entry is no page of the cache: nothing
// may be read or written there.  Offsets stay in 64 bits: a page's number times its size passes 32 bits in a long cache.
FT_PAGED_FN long long paged_page(const PagedTable& t, long long b, long long position) {
  if (position < 0) return -1;
  const long long col = position >> t.shift;
  if (col >= t.cols) return -1;
  const long long page = t.table[b * t.stride + col];
  return page >= 0 && page < t.n_pages ? page : -1;
}
FT_PAGED_FN long long paged_row(const PagedTable& t, long long position) {
  return position & ((1ll << t.shift) - 1);
}
// Tokens that a sequence has, of those that its table can hold; `bad` where the length says otherwise.
FT_PAGED_FN long long paged_length(const PagedTable& t, long long length, bool& bad) {
  const long long most = t.cols << t.shift;
  bad = length < 0 || length > most;
  return length < 0 ? 0 : (length > most ? most : length);
}

}  // namespace ftk
