// A paged key-value cache and the sequences of a step, as the kernels on them see both (include/krn_amd.h describes the
// layout). What lies on the device is checked on the device: token ranges are cut to the tokens there are, a length to the
// pages that the table has room for, and a page number outside of the cache reads as zeros and is never written.
#pragma once
#include "common.h"

namespace krn {

struct CacheView {
  const void *keys, *values;  // (pages, kv_heads, page, d) of 16-bit elements
  int64_t pages;
  int kv_heads, page_shift;   // a page holds 2^page_shift keys, 16 or more
};

struct SequencesView {
  const int *starts, *lengths, *table;  // (n + 1) or none, (n), (n, width)
  int n, width, step, tokens;           // without starts every sequence has `step` tokens
};

// The tokens of sequence i
struct TokenRange {
  int first, count;
};
__device__ __forceinline__ TokenRange token_range(const SequencesView& s, int i) {
  if (!s.starts) return {i * s.step, s.step};
  const int first = min(max(s.starts[i], 0), s.tokens), end = min(max(s.starts[i + 1], first), s.tokens);
  return {first, end - first};
}

// The length of sequence i, which positions count from, and how many of its keys the table can hold
__device__ __forceinline__ int sequence_length(const SequencesView& s, int i) { return max(s.lengths[i], 0); }
__device__ __forceinline__ int held_keys(const SequencesView& s, int length, int page_shift) {
  return (int)min((int64_t)length, (int64_t)s.width << page_shift);
}

}  // namespace krn

// Host side: what every entry point on a cache checks; false leaves a message.
struct CacheArguments {
  const char* name;
  int kind;
  const void *keys, *values, *starts, *lengths, *table;
  int64_t tokens, heads, kv_heads, d, pages, page, step, sequences, width;
};
bool krn_cache_arguments(const CacheArguments& a, krn::CacheView& cache, krn::SequencesView& sequences);
