// Keys and values in the pages of a cache, and the keeping of the pages: what the kernels and their host side share.
#pragma once

#include "sb_common.cuh"

namespace sb {

// Keys or values of a cache: (layers, pages, heads, slots, head_dim); strides in elements (append) or bytes (fork, compact).
struct CacheRef {
  char *ptr;
  long long sl, sp, sh, st;
};

// x / d for 0 <= x < 2^31 by a multiplication: with 2^l >= d > 2^(l - 1), the quotient is exactly x * ceil(2^(31 + l) / d) >> 31 + l.
struct FastDiv {
  unsigned mul;
  int post, one;
  __host__ static FastDiv by(int d) {
    int l = 0;
    while ((1LL << l) < d) ++l;
    return FastDiv{(unsigned)(((1ULL << (31 + l)) + d - 1) / d), l - 1, d == 1};
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int of(int x) const { return one ? x : (int)(__umulhi((unsigned)x, mul) >> post); }
#endif
};

struct AppendParams {
  TensorRef k, v;                  // (batch, heads, tokens, head_dim); packed: batch 1
  CacheRef kc, vc;                 // strides in elements
  const int *page_table;
  long long table_stride;
  const int *seq_lens;
  const void *cu;                  // packed: num_seq sequence ends; null: every sequence has `tokens` new tokens
  int cu64, check_leading_zero;
  int num_seq, kv_heads, head_dim, page_size, num_pages, max_pages, esize;
  long long tokens;                // of a sequence; packed: of all
  int per_block;                   // tokens of a block
  int per_row, per_token;          // copies of a row; of a token's rows, keys and values
  FastDiv by_row, by_token;
  int *status;
};

// The tables of a pool: which pages a sequence has, how long it is, how many sequences have a page.
struct PagesParams {
  int *page_table;
  long long table_stride;
  int *seq_lens, *refs;
  int max_seqs, max_pages, num_pages, page_size;
  const int *a, *b;                // extend: counts (or null); fork: sources, destinations; free: sequences
  int n, count;                    // entries of a and b; extend without counts: new tokens of every sequence that has some
  CacheRef k, v;                   // fork, compact: strides in bytes
  int layers, heads, row_bytes, vec;
  int per_row, parts, part_heads;  // copies of a row; a page's heads are copied by `parts` blocks, part_heads each
  FastDiv by_row, by_parts;
  int *work;                       // see pages_work_ints
  int *status;
};

// Scratch of the keeping operators, in ints: header, then one entry per page twice, one per sequence and pair each.
constexpr int kPagesHeader = 16;
inline long long pages_work_ints(long long num_pages, long long max_seqs, long long n) {
  return kPagesHeader + 2 * num_pages + max_seqs + 2 * n + 64;
}

cudaError_t launch_append(const AppendParams &p, cudaStream_t s);
cudaError_t launch_extend(const PagesParams &p, cudaStream_t s);
cudaError_t launch_fork(const PagesParams &p, cudaStream_t s, int *launches);
cudaError_t launch_free(const PagesParams &p, cudaStream_t s);
cudaError_t launch_compact(const PagesParams &p, cudaStream_t s, int *launches);

}  // namespace sb
