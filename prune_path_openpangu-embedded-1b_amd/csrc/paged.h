// What the paged-cache kernels share: the description of a ragged batch and its cache.
//
// n_seqs sequences; the rows cu_q[s] .. cu_q[s + 1] of the packed token axis are the new tokens of
// sequence s, and kv_lens[s] tokens are in the cache once they are appended, so row i of the
// sequence sits at position kv_lens[s] - (its new tokens) + i. Position p is in page
// block_table[s][p / page_size], place p % page_size. An entry outside [0, num_pages) and a
// position beyond the table (or below zero) hold no token: nothing is written there, nothing is
// attended there. Rows behind cu_q[n_seqs] belong to no sequence; the kernels treat them as
// sequence number n_seqs, of length 0.
#pragma once
#include "pp_common.h"

// Two floats rounded to bf16 and packed, a in the low half: one v_cvt_pk_bf16_f32.
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t f32_to_bf16x2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t));
}

struct PagedSeqs {
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* table;
  int n_rows, n_seqs;
  int max_pages, num_pages;
  int lp;  // log2 of the page size
  __device__ int start(int s) const {  // first row of sequence s, whatever the caller's array holds
    if (s <= 0) return 0;
    if (s > n_seqs) return n_rows;
    return min(max(cu_q[s], 0), n_rows);
  }
  // the page that an entry of the table names, -1 for none
  __device__ int page(int entry) const { return (unsigned)entry < (unsigned)num_pages ? entry : -1; }
  // positions that the table has room for
  __device__ int capacity() const { return max_pages << lp; }  // at most 2^30 (checked by the host)
};

// The loads above are not moved below this line, to where their values are used.
__device__ __forceinline__ void paged_asked() { asm volatile("" ::: "memory"); }

// The sequence that work item t belongs to, where sequence s has the items first(start(s), s)
// and on: the last s with first(start(s), s) <= t. `first` grows with s, by at least the items that
// the sequence has, so the item space needs no prefix sum. Every wave finds it for itself, 256
// sequences at a time: offsets and lengths come in one round of loads, and those of the sequence
// found are taken from the lanes that have them. s is in [0, n_seqs], also for offsets out of order;
// the rows of no sequence are number n_seqs, of length 0.
struct PagedSeq {
  int s, c0, rows;  // its number, its first row, how many rows
  int len;          // its tokens in the cache
};
template <typename F>
__device__ __forceinline__ PagedSeq paged_find(const PagedSeqs& q, int64_t t, F first) {
  const int lane = threadIdx.x & 63;
  int n = 0, s0 = 0;
  int c[4], k[4];
  const int32_t* const lens = q.n_seqs ? q.kv_lens : q.cu_q;  // (of no sequence: an address that can be read)
  for (;; s0 += 256) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // no branches: all eight loads are on their way together
      const int s = s0 + 64 * i + lane;
      c[i] = q.cu_q[min(s, q.n_seqs)];
      k[i] = lens[max(min(s, q.n_seqs - 1), 0)];
    }
    paged_asked();
    int m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + 64 * i + lane;
      c[i] = s == 0 ? 0 : s > q.n_seqs ? q.n_rows : min(max(c[i], 0), q.n_rows);
      k[i] = s < q.n_seqs ? k[i] : 0;
      m += __popcll(__ballot(s <= q.n_seqs && first(c[i], s) <= t));
    }
    n += m;
    if (m < 256 || s0 + 256 > q.n_seqs) break;
  }
  PagedSeq f;
  f.s = __builtin_amdgcn_readfirstlane(max(n - 1, 0));
  const int at = f.s - s0;  // < 0: the last of the 256 before
  auto pick = [](const int (&v)[4], int j) {
    const int x = j < 64 ? v[0] : j < 128 ? v[1] : j < 192 ? v[2] : v[3];
    return __builtin_amdgcn_readlane(x, j & 63);
  };
  f.c0 = at >= 0 ? pick(c, at) : __builtin_amdgcn_readfirstlane(q.start(f.s));
  f.len = at >= 0 ? pick(k, at) : __builtin_amdgcn_readfirstlane(q.kv_lens[f.s]);
  f.rows = max((at >= -1 && at < 255 ? pick(c, at + 1) : __builtin_amdgcn_readfirstlane(q.start(f.s + 1))) - f.c0, 0);
  return f;
}

static inline int paged_log2(int v) {
  for (int b = 0; b < 31; ++b)
    if ((1 << b) == v) return b;
  return -1;
}

// Checks of the sizes, and of all the arguments, that the append and the attention have in common.
int pp_paged_sizes(const char* what, int64_t n_tokens, int n_seqs, int max_pages, int num_pages, int page_size, int Hq,
                   int Hkv, int D);
int pp_paged_check(const char* what, int64_t n_tokens, int n_seqs, const void* cu_q, const void* kv_lens,
                   const void* block_table, int max_pages, const void* k_pages, const void* v_pages, int num_pages,
                   int page_size, int Hq, int Hkv, int D);
