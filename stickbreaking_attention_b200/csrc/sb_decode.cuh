// Attention of new tokens over a paged key-value cache: what its kernels share.
//
// A run of keys is summed up, per query row, by (o, L): o = sum of a_j v_j with the stick whole at the newest end of the run,
// L = log2 of the stick that is left at its oldest end.  Two neighbouring runs join to (o_new + 2^L_new o_old, L_new + L_old),
// and this is associative, so the cache of a sequence can be cut anywhere.
//
// An item is (sequence, key head, block of query rows); its keys are counted in units of one tile, 16 keys (or, in huge
// batches, of so many that 31 bits count them).  The units of all items lie one behind the other on one axis, which is cut into equal chunks, one per WARP of the grid: a batch of ragged lengths is
// spread evenly whatever the lengths are, only the device has to know them, and no warp ever waits for another.  A warp walks
// through the pieces of its chunk without a pause: its loads run a ring of stages ahead of its arithmetic and go on into the next
// piece while the last one's results are being written.  (With a block per chunk, its warps joined behind every piece, a piece
// cost 8 us more than its bytes: 64 sequences x 16 heads x 512..4096 keys 201 us, 24 short ones with 4 new tokens 60 us.)
//
// An item that a cut goes through leaves a piece per chunk in the workspace (two slots per chunk) for the join kernel, and a
// note of where they are.
#pragma once

#include "sb_common.cuh"

namespace sb {

constexpr int kTileKeys = 16;
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
  int items_per_seq;      // kv_heads * row_blocks
  int page_shift;         // page_size = 1 << page_shift, or -1: then key / page_size = (key * page_magic >> 32) >> page_post
  unsigned page_magic;
  int page_post;
  int attend_current, dense;
  int unit_shift;         // a unit is 1 << unit_shift keys
  float scale;
  int chunks;             // warps of the main kernel
  int by_item;            // notes are numbered by item, where there are fewer items than chunks; else by chunk
  float *part_o, *part_l; // per slot (2 * chunks of them): rows_per_block x part_cols sums, rows_per_block x L
  int part_cols;
  int4 *notes;            // [min(items, chunks)]: an item that was cut: sequence, item of it, first chunk, pieces (0: none)
  int *status;
};

// What a sequence's length says: its keys that some query attends to, or -1 for a length that cannot be.
__device__ __forceinline__ int seq_keys(const DecodeParams &p, int b) {
  const int len = p.seq_lens[b];
  if (!cached_length_ok(len, p.max_pages, p.page_size)) return -1;
  return max(len - (p.attend_current ? 0 : 1), 0);
}
__device__ __forceinline__ int units_of(const DecodeParams &p, int keys) {
  return keys <= 0 ? 1 : (int)(((unsigned)keys + (1u << p.unit_shift) - 1) >> p.unit_shift);
}
__device__ __forceinline__ int page_index(const DecodeParams &p, int key) {
  return p.page_shift >= 0 ? key >> p.page_shift : (int)(__umulhi((unsigned)key, p.page_magic) >> p.page_post);
}
// Keys that query row r (= head of the group * new_tokens + token) attends to are those before this one.
__device__ __forceinline__ int row_limit(const DecodeParams &p, int keys, int r) {
  return p.new_tokens == 1 ? keys : max(keys - (p.new_tokens - 1 - r % p.new_tokens), 0);
}

// One chunk's part of one item: keys [k0, k1) for the query rows [row0, row0 + rows) of key head `head`.
struct Piece {
  int seq, head, row0, rows, keys, k0, k1;
  int edge;               // some row does not attend to the keys from here on (k1 and more if there is no such row)
};

// Where a chunk is on its way through the items.
struct Cursor {
  int seq, item, u0, n, keys;   // item of the sequence, unit of the item, units of every item of the sequence, seq_keys
  int rest;                     // units from here to the chunk's end
  __device__ __forceinline__ void read_seq(const DecodeParams &p) {
    keys = seq_keys(p, seq);
    n = units_of(p, keys);
  }
  __device__ __forceinline__ int count() const { return min(n - u0, rest); }
  __device__ __forceinline__ void advance(const DecodeParams &p) {
    rest -= count();
    u0 = 0;
    if (++item == p.items_per_seq) {
      item = 0;
      ++seq;
      if (rest > 0) read_seq(p);
    }
  }
  __device__ __forceinline__ Piece piece(const DecodeParams &p) const {
    Piece w;
    w.seq = seq;
    w.keys = max(keys, 0);
    w.head = p.row_blocks == 1 ? item : item / p.row_blocks;
    w.row0 = (item - w.head * p.row_blocks) * p.rows_per_block;
    w.rows = min(p.rows - w.row0, p.rows_per_block);
    // the first and the last token among the rows: what none of them attends to is not read, what some do not is looked at per row
    const int tok = p.new_tokens == 1 ? 0 : w.row0 % p.new_tokens, last = tok + w.rows - 1;
    const int high = min(last, p.new_tokens - 1), low = last >= p.new_tokens ? 0 : tok;
    w.k0 = u0 << p.unit_shift;
    w.k1 = max(min(u0 + count() == n ? w.keys : (u0 + count()) << p.unit_shift, w.keys - (p.new_tokens - 1 - high)), w.k0);
    w.edge = w.keys - (p.new_tokens - 1 - low);
    return w;
  }
};
__device__ __forceinline__ int tiles_of(const Piece &w) { return (w.k1 - w.k0 + kTileKeys - 1) / kTileKeys; }

// The block's warps' chunks: warp w has chunk w * blocks + block, so that few units are spread over many SMs.  By all threads
// of the block; contains barriers.
template <int kWarps> struct ChunkShared {
  int sum[kWarps], before[kWarps * 32 + 1];    // units of each warp's sequences; units before each thread's
};
template <int kWarps>
__device__ __forceinline__ Cursor find_chunk(const DecodeParams &p, int &chunk, int &size, ChunkShared<kWarps> &shared) {
  constexpr int kThreads = kWarps * 32;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int each = (p.batch + kThreads - 1) / kThreads, b0 = min(t * each, p.batch), b1 = min(b0 + each, p.batch);
  int own = 0;
  for (int b = b0; b < b1; ++b) own += p.items_per_seq * units_of(p, seq_keys(p, b));
  int sum = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += other;
  }
  if (lane == 31) shared.sum[warp] = sum;
  __syncthreads();
  int before = sum - own, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += shared.sum[w];
    total += shared.sum[w];
  }
  shared.before[t] = before;
  if (t == 0) shared.before[kThreads] = total;
  __syncthreads();
  size = (total - 1) / p.chunks + 1;
  chunk = warp * gridDim.x + blockIdx.x;
  Cursor c;
  c.rest = c.seq = c.item = c.u0 = c.n = c.keys = 0;
  if ((long long)chunk * size >= total) return c;
  const int unit = chunk * size;
  c.rest = min(size, total - unit);
  int group = 0;                               // the warp, then the thread, whose units this one is among
#pragma unroll
  for (int w = 1; w < kWarps; ++w)
    if (shared.before[32 * w] <= unit) group = 32 * w;
  const uint32_t vote = __ballot_sync(0xffffffffu, shared.before[group + lane] <= unit && shared.before[group + lane + 1] > unit);
  const int owner = group + __ffs(vote) - 1;
  int first = shared.before[owner];
  for (c.seq = owner * each;; ++c.seq) {
    c.read_seq(p);
    const int all = p.items_per_seq * c.n;
    if (unit - first < all) break;
    first += all;
  }
  c.item = (unit - first) / c.n;
  c.u0 = unit - first - c.item * c.n;
  return c;
}

__device__ __forceinline__ long long row_offset(const DecodeParams &p, const TensorRef &t, int seq, int head, int row) {
  const int g = p.new_tokens == 1 ? row : row / p.new_tokens, tok = row - g * p.new_tokens;
  return seq * t.sb + (head * (long long)(p.heads / p.kv_heads) + g) * t.sh + tok * t.st;
}
__device__ __forceinline__ long long rem_index(const DecodeParams &p, int seq, int head, int row) {
  const int g = p.new_tokens == 1 ? row : row / p.new_tokens, tok = row - g * p.new_tokens;
  return ((long long)seq * p.heads + head * (p.heads / p.kv_heads) + g) * p.new_tokens + tok;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

// A warp's loads, newest tile of a piece first, on into the next pieces.  32 entries of the page table are kept in a register of
// the warp and read anew, ahead of their use, where a tile needs others.
template <typename E> struct Feed {
  const DecodeParams &p;
  Cursor c;
  Piece w;
  int left = 0, number = 0;     // tiles of the piece that are still to be copied; how many pieces came before it
  int window = 0, top = -1;     // lane l has entry top - l of the sequence's row
  uint32_t bad = 0;             // a bit per stage: a page that is none

  __device__ __forceinline__ Feed(const DecodeParams &p_, const Cursor &at) : p(p_), c(at) { open(); }
  __device__ __forceinline__ void open() {
    top = -1;
    if (c.rest == 0) return;
    w = c.piece(p);
    left = tiles_of(w);
    E::prefetch_rows(p, w);
  }
  // By all lanes, before each copy but ahead of the one before it: the next tile's pages.
  __device__ __forceinline__ void seek() {
    while (left == 0) {
      if (c.rest == 0) return;
      c.advance(p);
      ++number;
      open();
    }
    const int key0 = w.k0 + (left - 1) * kTileKeys;
    const int low = page_index(p, key0);
    if (top < 0 || low < top - 31) {
      top = page_index(p, min(key0 + kTileKeys, w.k1) - 1);
      const int entry = top - (int)(threadIdx.x & 31);
      window = entry >= 0 ? p.page_table[w.seq * p.table_stride + entry] : -1;
    }
  }
  // Lane l's key of the tile (l & 15): its page, -1 for none, and whether it should have one.
  __device__ __forceinline__ int page_of(int key) {
    const int page = __shfl_sync(0xffffffffu, window, top - page_index(p, min(key, w.k1 - 1)));
    return (unsigned)page < (unsigned)p.num_pages ? page : -1;
  }
  __device__ __forceinline__ void copy(int stage, char *to) {
    if (left == 0) return;
    const int key0 = w.k0 + --left * kTileKeys;
    bool wrong;
    if (p.page_shift >= 4 && key0 + kTileKeys <= w.k1) {          // a whole tile in one page
      const int page = page_of(key0);
      wrong = page < 0;
      if (!wrong) E::copy_run(p, w, page, key0 & ((1 << p.page_shift) - 1), to);
      else E::copy(p, w, -1, 0, to);
    } else {
      const int key = key0 + (threadIdx.x & 15);
      int page = page_of(key);
      wrong = __any_sync(0xffffffffu, page < 0);
      if (key >= w.k1) page = -1;
      E::copy(p, w, page, key - page_index(p, key) * p.page_size, to);
    }
    if (wrong && (threadIdx.x & 31) == 0 && p.status != nullptr) {
      p.status[0] = SB_DEV_BAD_PAGE;
      p.status[1] = w.seq;
    }
    bad = (bad & ~(1u << stage)) | (uint32_t)wrong << stage;
    seek();
  }
  // what is left of piece `which` is not wanted; how many of its tiles that is
  __device__ __forceinline__ int drop(int which) {
    if (number != which || left == 0) return 0;
    const int dropped = left;
    left = 0;
    seek();
    return dropped;
  }
};

// The main kernel.  E, the engine: the shape of a stage (kWarps, kStages, kStage bytes), copy (16 keys and values of one
// key head), start, tile (adds a stage up, keys newest first), gone (the rows' sticks are used up), finish (writes the sums out).
// One loop and one place for each of these: a short call runs through the code once, and its length counts there.
template <typename E> __device__ __forceinline__ void decode_chunks(const DecodeParams &p, char *memory, ChunkShared<E::kWarps> &shared) {
  int chunk, size;
  Cursor c = find_chunk<E::kWarps>(p, chunk, size, shared);
  const int lane = threadIdx.x & 31;
  if (!p.by_item && lane == 0) p.notes[chunk] = make_int4(0, 0, 0, 0);
  if (c.rest == 0) return;
  char *stages = memory + (threadIdx.x >> 5) * E::kStages * E::kStage;
  Feed<E> feed(p, c);
  feed.seek();
  Piece w;
  E sum;
  int at = 0, into = 0, fill = E::kStages, number = 0, left = 0;
  bool fresh = true, bad = false, done = false, first = true;
  for (;;) {
    if (fill > 0) {              // a stage is free
      __syncwarp();
      feed.copy(into, stages + into * E::kStage);
      cp_async_commit();
      into = into == E::kStages - 1 ? 0 : into + 1;
      if (--fill > 0) continue;
    }
    if (fresh) {
      w = c.piece(p);
      sum.start(p, w);
      left = tiles_of(w);
      bad = c.keys < 0;
      fresh = done = false;
    }
    if (left > 0) {
      cp_async_wait<E::kStages - 1>();
      __syncwarp();
      if (!done) {
        bad |= feed.bad >> at & 1;
        sum.tile(p, w, stages + at * E::kStage, w.k0 + (left - 1) * kTileKeys);
        if (!p.dense && sum.gone()) {
          done = true;           // the tiles that are on their way still come by
          left -= feed.drop(number);
        }
      }
      --left;
      at = at == E::kStages - 1 ? 0 : at + 1;
      fill = 1;
    }
    if (left > 0) continue;
    const int count = c.count();
    const bool whole = c.u0 == 0 && count == c.n;
    sum.finish(p, w, whole ? -1 : 2 * chunk + (first && c.u0 > 0 ? 0 : 1), bad);
    if (lane == 0) {
      if (c.u0 == 0) {
        const int pieces = whole ? 0 : 1 + (c.n - count + size - 1) / size;
        if (p.by_item) p.notes[c.seq * p.items_per_seq + c.item] = make_int4(c.seq, c.item, chunk, pieces);
        else if (!whole) p.notes[chunk] = make_int4(c.seq, c.item, chunk, pieces);
      }
      if (c.keys < 0 && p.status != nullptr) {
        p.status[0] = SB_DEV_BAD_SEQ_LEN;
        p.status[1] = c.seq;
      }
    }
    c.advance(p);
    if (c.rest == 0) break;
    ++number;
    first = false;
    fresh = true;
  }
  cp_async_wait<0>();
}

// Where row r of a piece's result goes: to o and rem where the piece is the whole item, else to its slot of the workspace.
template <typename T> struct RowOut {
  T *o;
  float *part;
  __device__ __forceinline__ RowOut(const DecodeParams &p, const Piece &w, int slot, int r) {
    o = reinterpret_cast<T *>(p.o.ptr) + row_offset(p, p.o, w.seq, w.head, w.row0 + r);
    part = slot < 0 ? nullptr : p.part_o + ((long long)slot * p.rows_per_block + r) * p.part_cols;
  }
  __device__ __forceinline__ void put(int col, float x) const {
    if (part == nullptr) o[col] = from_f32<T>(x);
    else part[col] = x;
  }
};
template <typename T> __device__ __forceinline__ void put_rem(const DecodeParams &p, const Piece &w, int slot, int r, float left) {
  if (slot < 0)
    reinterpret_cast<T *>(p.rem)[rem_index(p, w.seq, w.head, w.row0 + r)] = from_f32<T>(exp2f(left));
  else
    p.part_l[(long long)slot * p.rows_per_block + r] = left;
}
// The rows of q that a piece will want: on their way to L2 while the piece before it is worked on.
__device__ __forceinline__ void prefetch_q(const DecodeParams &p, const Piece &w, int esize) {
  const int lane = threadIdx.x & 31;
  if (lane >= w.rows) return;
  const char *row = p.q.ptr + row_offset(p, p.q, w.seq, w.head, w.row0 + lane) * esize;
  for (int at = 0; at < p.head_dim * esize; at += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + at));
}

// 2^x down to the smallest numbers (ptx::ex2 gives 0 for what is below 2^-126; weights go down to 2^-149, where a stick counts as
// used up), to 2^-22 of itself.
__device__ __forceinline__ float exp2_all(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A sum of many terms in 32 bits whose rounding errors are kept and added to the next term.
struct LongSum {
  float sum = 0.0f, lost = 0.0f;
  __device__ __forceinline__ void add(float x) {
    const float y = x + lost, s = sum + y;
    lost = isinf(s) ? 0.0f : y - (s - sum);
    sum = s;
  }
};

cudaError_t launch_decode_simt(const DecodeParams &p, int dtype, cudaStream_t s);
cudaError_t launch_decode_tc(const DecodeParams &p, int dtype, cudaStream_t s);
cudaError_t launch_decode_join(const DecodeParams &p, int dtype, cudaStream_t s);      // of the CUDA-core kernel's pieces
cudaError_t launch_decode_tc_join(const DecodeParams &p, int dtype, cudaStream_t s);
int decode_tc_rows(int rows, int head_dim);     // query rows per item
int decode_simt_rows(int rows, int head_dim);
int decode_tc_cols(int head_dim);               // columns of a piece in the workspace
int decode_tc_warps(int rows, int head_dim);    // warps per block for so many rows per item; one block per SM
int decode_simt_warps(int rows, int head_dim);

}  // namespace sb
