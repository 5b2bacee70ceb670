// Attention of new tokens over a paged key-value cache: what its kernels share.
//
// A run of keys is summed up, per query row, by (o, L): o = sum of a_j v_j with the stick whole at the newest end of the run,
// L = log2 of the stick that is left at its oldest end.  Two neighbouring runs join to (o_new + 2^L_new o_old, L_new + L_old),
// and this is associative, so the cache of a sequence can be cut anywhere: into pieces for blocks, into ranges for warps.
//
// An item is (sequence, key head, block of query rows); its keys are counted in units of kUnit.  The units of all items lie
// one behind the other on one axis, which is cut into equal chunks, one per block: a batch of ragged lengths is spread evenly
// whatever the lengths are, and only the device has to know them.  An item that a cut goes through leaves a piece per block in
// the workspace (two slots per block) for the join kernel.
#pragma once

#include "sb_common.cuh"

namespace sb {

constexpr int kUnit = 64;
// A weight below 2^-150 is exactly 0 in fp32, the smallest of whose numbers is 2^-149.
constexpr float kStickGone = -150.0f;

struct PagedRef {
  const char *ptr;
  long long sp, sh, st;   // element strides of page, head, slot
};

struct DecodeParams {
  TensorRef q, o;
  char *rem;              // (batch, heads, new_tokens) contiguous
  PagedRef k, v;
  const int *page_table;
  long long table_stride;
  const int *seq_lens;
  int batch, heads, kv_heads, new_tokens, head_dim, page_size, num_pages, max_pages;
  int rows, row_blocks, rows_per_block;   // query rows of a key head = heads / kv_heads * new_tokens, and how they are cut
  int attend_current, dense;
  float scale;
  int chunks, min_units;  // blocks of the main kernel; units that a block takes at least
  float *part_o, *part_l; // [2 * chunks][rows_per_block][head_dim], [2 * chunks][rows_per_block]
  int *status;
};

// What a sequence's length says: its keys that some query attends to, or -1 for a length that cannot be.
__device__ __forceinline__ int seq_keys(const DecodeParams &p, int b) {
  const int len = p.seq_lens[b];
  if (len < 0 || len > (long long)p.max_pages * p.page_size) return -1;
  return max(len - (p.attend_current ? 0 : 1), 0);
}
__device__ __forceinline__ int units_of(int keys) { return max((max(keys, 0) + kUnit - 1) / kUnit, 1); }
// Keys that query row r (= head of the group * new_tokens + token) attends to are those before this one.
__device__ __forceinline__ int row_limit(const DecodeParams &p, int keys, int r) {
  return max(keys - (p.new_tokens - 1 - r % p.new_tokens), 0);
}

struct Place {            // a position on the axis of units
  long long units, chunk; // of the whole axis, and per block
  int seq;
  long long first;        // where the units of `seq` begin
};

// By all threads of the block (a multiple of 32, at most 1024); contains barriers.  Where unit `chunk_index * chunk + shift`
// lies.  `shared`: 40 long longs.
template <int kThreads>
__device__ __forceinline__ Place find_place(const DecodeParams &p, int chunk_index, int shift, long long *shared) {
  const int per_item = p.kv_heads * p.row_blocks, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int each = (p.batch + kThreads - 1) / kThreads, b0 = min(t * each, p.batch), b1 = min(b0 + each, p.batch);
  long long own = 0;
  for (int b = b0; b < b1; ++b) own += (long long)per_item * units_of(seq_keys(p, b));
  long long sum = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += other;
  }
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = total;
    total += shared[w];
  }
  before += sum - own;
  Place at;
  at.units = total;
  at.chunk = max((total + p.chunks - 1) / p.chunks, (long long)p.min_units);
  const long long unit = chunk_index * at.chunk + shift;
  if (unit >= before && unit < before + own) {
    int b = b0;
    for (;; ++b) {
      const long long n = (long long)per_item * units_of(seq_keys(p, b));
      if (unit < before + n) break;
      before += n;
    }
    shared[32] = b;
    shared[33] = before;
  }
  __syncthreads();
  at.seq = (int)shared[32];
  at.first = shared[33];
  return at;
}

// One block's part of one item: keys [k0, k1) for the query rows [row0, row0 + rows) of key head `head`.
struct Piece {
  int seq, head, row0, rows, keys, k0, k1;
  int edge;               // some row does not attend to the keys from here on (k1 and more if there is no such row)
  int slot;               // where it is left for the join kernel, -1: it is the whole item
  bool bad;               // the sequence's length was refused
};

// The piece at `unit` of a block's units [.., end); returns the units it takes.
__device__ __forceinline__ int next_piece(const DecodeParams &p, const Place &at, int chunk_index, long long unit, long long begin,
                                          long long end, int keys, Piece &w) {
  w.bad = keys < 0;
  w.keys = max(keys, 0);
  const int n = units_of(keys);
  const long long in_seq = unit - at.first;
  const int item = (int)(in_seq / n), u0 = (int)(in_seq - (long long)item * n);
  const int count = (int)min((long long)(n - u0), end - unit);
  w.seq = at.seq;
  w.head = item / p.row_blocks;
  w.row0 = (item - w.head * p.row_blocks) * p.rows_per_block;
  w.rows = min(p.rows - w.row0, p.rows_per_block);
  // the first and the last token among the rows: what none of them attends to is not read, what some do not is looked at per row
  const int tok = w.row0 % p.new_tokens, last = tok + w.rows - 1;
  const int high = min(last, p.new_tokens - 1), low = last >= p.new_tokens ? 0 : tok;
  w.k0 = u0 * kUnit;
  w.k1 = max(min((u0 + count) * kUnit, w.keys - (p.new_tokens - 1 - high)), w.k0);
  w.edge = w.keys - (p.new_tokens - 1 - low);
  const bool whole = u0 == 0 && count == n;
  w.slot = whole ? -1 : 2 * chunk_index + (u0 > 0 && unit == begin ? 0 : 1);
  return count;
}

__device__ __forceinline__ long long row_offset(const DecodeParams &p, const TensorRef &t, const Piece &w, int r) {
  const int row = w.row0 + r, g = row / p.new_tokens, tok = row - g * p.new_tokens;
  return w.seq * t.sb + (w.head * (long long)(p.heads / p.kv_heads) + g) * t.sh + tok * t.st;
}
__device__ __forceinline__ long long rem_index(const DecodeParams &p, const Piece &w, int r) {
  const int row = w.row0 + r, g = row / p.new_tokens, tok = row - g * p.new_tokens;
  return ((long long)w.seq * p.heads + w.head * (p.heads / p.kv_heads) + g) * p.new_tokens + tok;
}

// The page that holds a key, or -1 (and the status word) for an entry of the table that is none.
__device__ __forceinline__ int page_of(const DecodeParams &p, int seq, int index) {
  const int page = p.page_table[seq * p.table_stride + index];
  if ((unsigned)page < (unsigned)p.num_pages) return page;
  if (p.status != nullptr) {
    p.status[0] = SB_DEV_BAD_PAGE;
    p.status[1] = seq;
  }
  return -1;
}

// The epilogue of a piece, by all threads of the block behind a barrier: joins the warps' sums (warp 0 has the newest keys),
// warp n's at sums + n * warp_stride as [rows][width] times `unscale`, and writes the result or leaves it for the join kernel.
template <typename T, int kThreads, int kWarps, int kRows>
__device__ __forceinline__ void finish_piece(const DecodeParams &p, const Piece &w, const float *sums, int warp_stride, int width,
                                             float unscale, const float (&left_of)[kWarps][kRows]) {
  for (int e = threadIdx.x; e < w.rows * p.head_dim; e += kThreads) {
    const int r = e / p.head_dim, c = e - r * p.head_dim;
    float o = 0.0f, left = 0.0f;
    for (int n = 0; n < kWarps; ++n) {
      const float stick = exp2f(left);
      if (stick == 0.0f) break;
      o += stick * sums[n * warp_stride + r * width + c];
      left += left_of[n][r];
    }
    o *= unscale;
    if (w.slot < 0)
      reinterpret_cast<T *>(p.o.ptr)[row_offset(p, p.o, w, r) + c] = from_f32<T>(o);
    else
      p.part_o[((long long)w.slot * p.rows_per_block + r) * p.head_dim + c] = o;
  }
  for (int r = threadIdx.x; r < w.rows; r += kThreads) {
    float left = 0.0f;
    for (int n = 0; n < kWarps; ++n) left += left_of[n][r];
    if (w.slot < 0)
      reinterpret_cast<T *>(p.rem)[rem_index(p, w, r)] = from_f32<T>(exp2f(left));
    else
      p.part_l[(long long)w.slot * p.rows_per_block + r] = left;
  }
  if (w.bad && threadIdx.x == 0 && p.status != nullptr) {
    p.status[0] = SB_DEV_BAD_SEQ_LEN;
    p.status[1] = w.seq;
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

cudaError_t launch_decode_simt(const DecodeParams &p, int dtype, cudaStream_t s);
cudaError_t launch_decode_join(const DecodeParams &p, int dtype, cudaStream_t s);
cudaError_t launch_decode_tc(const DecodeParams &p, int dtype, cudaStream_t s);
int decode_tc_rows(int rows, int head_dim);
int decode_simt_rows(int rows, int head_dim);   // query rows per item

}  // namespace sb
