// The pages of a key-value cache: new keys and values written into them, and their keeping (room for new tokens, forks, freed
// sequences, compaction) with the tables on the device, so that a serving step needs no host synchronisation and can be captured.
//
// Which page a sequence gets is a rule, not a race: the lowest free pages (count 0), in the order of sequences and positions.
// An operator that cannot do all it is asked to (too few pages, an index that is none, a length that cannot be) changes nothing and
// says so in the status word.  Entries of the table that name no page, or a free one, are found on the way by freeing and
// compaction: these are passed over, and reported.
#include "sb_pages.cuh"

#include <algorithm>
#include <initializer_list>

namespace sb {

namespace {

// ---- append -------------------------------------------------------------------------------------------------------------
// Memory-bound: every new row read and written once.  A block looks up where its tokens go (sequence, page, slot), then its
// threads copy 16 bytes at a time, all heads of a token, keys and values, kDeep of them in flight per thread.
constexpr int kAppendThreads = 256, kMaxTokens = 64, kAppendBlocks = 32;

__device__ __forceinline__ long long append_end(const AppendParams &p, int i) {
  return p.cu64 ? reinterpret_cast<const long long *>(p.cu)[i] : (long long)reinterpret_cast<const int *>(p.cu)[i];
}
__device__ __forceinline__ void report(int *status, int code, int which) {
  if (status != nullptr) {
    status[0] = code;
    status[1] = which;
  }
}

template <typename V>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ long long src[kMaxTokens], dst[kMaxTokens];   // elements; of the keys' tensors, and of the values' in the loop
  __shared__ long long vsrc[kMaxTokens], vdst[kMaxTokens];
  enter_kernel<true>();
  if (p.cu != nullptr) {
    bool bad = false;
    for (int i = threadIdx.x; i < p.num_seq; i += kAppendThreads) {
      const long long start = i == 0 ? 0 : append_end(p, i - 1), end = append_end(p, i);
      if (start < 0 || end < start || end > p.tokens) {
        bad = true;
        if (blockIdx.x == 0) report(p.status, SB_DEV_BAD_CU_SEQLENS, i);
      }
    }
    if (p.check_leading_zero && threadIdx.x == 0 && append_end(p, -1) != 0) {
      bad = true;
      if (blockIdx.x == 0) report(p.status, SB_DEV_BAD_CU_SEQLENS, -1);
    }
    if (__syncthreads_or(bad)) return;
  }
  const long long all = p.cu != nullptr ? p.tokens : p.tokens * p.num_seq;
  const long long t0 = (long long)blockIdx.x * p.per_block;
  const int count = (int)min((long long)p.per_block, all - t0);
  if ((int)threadIdx.x < count) {
    const long long token = t0 + threadIdx.x;
    long long seq, back, from = token;        // back: how many tokens of the sequence follow, with this one
    if (p.cu != nullptr) {
      int lo = 0, hi = p.num_seq;             // the first sequence that ends behind the token
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (append_end(p, mid) > token) hi = mid;
        else lo = mid + 1;
      }
      seq = lo;
      back = lo < p.num_seq ? append_end(p, lo) - token : 0;
    } else {
      seq = token / p.tokens;
      from = token - seq * p.tokens;
      back = p.tokens - from;
    }
    long long to = -1;
    if (back > 0) {
      const int len = p.seq_lens[seq];
      const long long pos = len - back;
      if (!cached_length_ok(len, p.max_pages, p.page_size)) report(p.status, SB_DEV_BAD_SEQ_LEN, (int)seq);
      else if (pos >= 0) {
        const int index = (int)(pos / p.page_size), page = p.page_table[seq * p.table_stride + index];
        if ((unsigned)page >= (unsigned)p.num_pages) report(p.status, SB_DEV_BAD_PAGE, (int)seq);
        else {
          const int slot = (int)(pos - (long long)index * p.page_size);
          to = page * p.kc.sp + slot * p.kc.st;
          vdst[threadIdx.x] = page * p.vc.sp + slot * p.vc.st;
        }
      }
    }
    const long long b = p.cu != nullptr ? 0 : seq;
    src[threadIdx.x] = b * p.k.sb + from * p.k.st;
    vsrc[threadIdx.x] = b * p.v.sb + from * p.v.st;
    dst[threadIdx.x] = to;
  }
  __syncthreads();
  const int per_row = p.per_row, per_token = p.per_token, work = count * per_token;
  constexpr int kDeep = 4;
  for (int e0 = threadIdx.x; e0 < work; e0 += kDeep * kAppendThreads) {
    V x[kDeep];
    V *to[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int e = e0 + i * kAppendThreads;
      to[i] = nullptr;
      if (e < work) {
        const int t = p.by_token.of(e), in = e - t * per_token, row = p.by_row.of(in), c = in - row * per_row;
        const bool val = row >= p.kv_heads;
        const int h = val ? row - p.kv_heads : row;
        if (dst[t] >= 0) {
          const TensorRef &s = val ? p.v : p.k;
          const CacheRef &d = val ? p.vc : p.kc;
          x[i] = reinterpret_cast<const V *>(s.ptr + ((val ? vsrc[t] : src[t]) + h * s.sh) * p.esize)[c];
          to[i] = reinterpret_cast<V *>(d.ptr + ((val ? vdst[t] : dst[t]) + h * d.sh) * p.esize) + c;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (to[i] != nullptr) *to[i] = x[i];
  }
}

// ---- the keeping of the pages ----------------------------------------------------------------------------------------------
// One block decides what happens (which pages go where), many carry it out.  The deciding block reads the counts of all pages,
// 16 per thread at a time.  What it takes for a small pool is a chain of trips to memory and barriers, so its lists are in shared
// memory where they are short, and it has 256 threads where those do (a fork of 4 sequences in 160 pages took 4.0 us, 7.6 with
// 1024 and lists in the workspace; 5.1 with the look at the sources' rows).
constexpr int kBookThreads = 1024, kFewThreads = 256, kPer = 16, kShort = 2048;
struct Book {
  int scan[33];
  int list[kShort], other[kShort];
};
inline int book_threads(const PagesParams &p) {
  return p.num_pages <= kFewThreads * kPer && p.max_seqs <= 2 * kFewThreads && p.n <= 2 * kFewThreads ? kFewThreads : kBookThreads;
}

// Exclusive prefix sum over the block's threads; total in `all`.  shared: 33 ints.  Contains barriers.
__device__ __forceinline__ int block_scan(int x, int *shared, int &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += other;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    const int own = lane < (int)(blockDim.x >> 5) ? shared[lane] : 0;
    int s = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += other;
    }
    shared[lane] = s - own;
    if (lane == 31) shared[32] = s;
  }
  __syncthreads();
  all = shared[32];
  return shared[warp] + sum - x;
}

// The counts of the pages [first, first + kPer); -1 behind the last page.
__device__ __forceinline__ void read_refs(const PagesParams &p, int first, int (&x)[kPer]) {
  if (first + kPer <= p.num_pages && reinterpret_cast<uintptr_t>(p.refs) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const int4 v = *reinterpret_cast<const int4 *>(p.refs + first + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = first + i < p.num_pages ? p.refs[first + i] : -1;
  }
}

// The `want` lowest free pages, into list; false if there are fewer.
__device__ __forceinline__ bool list_free(const PagesParams &p, int want, int *list, int *shared) {
  int found = 0;
  for (int base = 0; base < p.num_pages && found < want; base += (int)blockDim.x * kPer) {
    const int first = base + threadIdx.x * kPer;
    int x[kPer], mine = 0, all;
    read_refs(p, first, x);
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += x[i] == 0;
    int rank = found + block_scan(mine, shared, all);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (x[i] == 0) {
        if (rank < want) list[rank] = first + i;
        ++rank;
      }
    found += all;
  }
  __syncthreads();
  return found >= want;
}

__device__ __forceinline__ bool length_ok(const PagesParams &p, long long len) { return cached_length_ok(len, p.max_pages, p.page_size); }
__device__ __forceinline__ int pages_for(const PagesParams &p, int len) { return (int)(((long long)len + p.page_size - 1) / p.page_size); }

// New tokens of sequence b.
__device__ __forceinline__ int extra(const PagesParams &p, int b, int len) { return p.a != nullptr ? p.a[b] : len > 0 ? p.count : 0; }

__global__ void __launch_bounds__(kBookThreads) extend_kernel(const __grid_constant__ PagesParams p) {
  __shared__ Book book;
  int *const shared = book.scan;
  enter_kernel<true>();
  int *list = p.work + kPagesHeader, *const prefix = p.max_seqs <= kShort ? book.other : list + p.num_pages;
  __shared__ unsigned long long needed;
  int want = 0;
  unsigned long long asked = 0;
  bool bad = false;
  if (threadIdx.x == 0) needed = 0;
  for (int base = 0; base < p.max_seqs; base += blockDim.x) {
    const int b = base + threadIdx.x;
    int need = 0;
    if (b < p.max_seqs) {
      const int len = p.seq_lens[b], more = extra(p, b, len);
      if (more < 0 || !length_ok(p, len) || !length_ok(p, (long long)len + more)) {
        bad = true;
        report(p.status, SB_DEV_BAD_SEQ_LEN, b);
      } else {
        need = pages_for(p, len + more) - pages_for(p, len);
        asked += need;
        need = min(need, p.num_pages + 1);
      }
    }
    int all;
    const int before = block_scan(need, shared, all);
    // (a sum beyond the pool is refused below; kept from wrapping here)
    if (b < p.max_seqs) prefix[b] = want + before;
    want = min(want + all, p.num_pages + 1);
  }
  if (__syncthreads_or(bad)) return;
  if (want <= kShort) list = book.list;
  if (want > 0 && !list_free(p, want, list, shared)) {
    atomicAdd(&needed, asked);
    __syncthreads();
    if (threadIdx.x == 0) report(p.status, SB_DEV_OUT_OF_PAGES, (int)min(needed, 0x7fffffffULL));
    return;
  }
  for (int r = threadIdx.x; r < want; r += blockDim.x) {
    int lo = 0, hi = p.max_seqs;              // the last sequence whose pages begin at or before r
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (prefix[mid] <= r) lo = mid;
      else hi = mid;
    }
    const int page = list[r];
    p.page_table[lo * p.table_stride + pages_for(p, p.seq_lens[lo]) + r - prefix[lo]] = page;
    p.refs[page] = 1;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.max_seqs; b += blockDim.x) {
    const int len = p.seq_lens[b], more = extra(p, b, len);
    if (more > 0) p.seq_lens[b] = len + more;
  }
}

// No count goes below 0: a page whose count would is taken out of the row, and reported.
constexpr int kFreeThreads = 128, kFreeBlocks = 8;
__device__ __forceinline__ void free_row(const PagesParams &p, int b, int len, int thread, int threads) {
  const int pages = pages_for(p, len);
  int *const row = p.page_table + b * p.table_stride;
  constexpr int kDeep = 4;
  for (int i0 = thread; i0 < pages; i0 += kDeep * threads) {
    int page[kDeep], count[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int i = i0 + k * threads;
      page[k] = 0;
      count[k] = i < pages ? 0 : 1;
      if (i < pages) {
        page[k] = row[i];
        row[i] = -1;
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (count[k] == 0 && (unsigned)page[k] < (unsigned)p.num_pages) {
        count[k] = atomicSub(p.refs + page[k], 1);
        if (count[k] <= 0) atomicAdd(p.refs + page[k], 1);
      }
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (count[k] <= 0) report(p.status, SB_DEV_BAD_PAGE, b);
  }
}
// A block per entry, or, where the entries are more than kFreeBlocks times the SMs, a warp for every so many.  Each block looks at the
// whole list first.  Nothing that it refuses changes meanwhile: a length that another block has made 0 was one that can be.
// A sequence that is listed more than once is the first entry's (blocks), or theirs who takes its length (warps: an atomic in the
// chain, which a short call feels by 0.5 us).  3000 sequences of 20 pages: 18.4 us, 29.6 with a block per entry; 65535 of 10: 280, 7440.
__global__ void __launch_bounds__(kFreeThreads) free_kernel(const __grid_constant__ PagesParams p) {
  enter_kernel<true>();
  const int own = p.a[blockIdx.x];
  bool leave = false, first = true;
  for (int i = threadIdx.x; i < p.n; i += kFreeThreads) {
    const int s = p.a[i], code = (unsigned)s >= (unsigned)p.max_seqs ? SB_DEV_BAD_SEQUENCE : length_ok(p, p.seq_lens[s]) ? 0 : SB_DEV_BAD_SEQ_LEN;
    leave |= code != 0;
    first &= s != own || i >= (int)blockIdx.x;
    if (code != 0 && blockIdx.x == 0) report(p.status, code, s);
  }
  const bool by_block = p.n == (int)gridDim.x;
  if (__syncthreads_or(leave || (by_block && !first))) return;
  if (by_block) {
    free_row(p, own, p.seq_lens[own], threadIdx.x, kFreeThreads);
    __syncthreads();
    if (threadIdx.x == 0) p.seq_lens[own] = 0;
    return;
  }
  constexpr int kWarps = kFreeThreads / 32;
  const int lane = threadIdx.x & 31;
  for (int e = blockIdx.x * kWarps + (threadIdx.x >> 5); e < p.n; e += gridDim.x * kWarps) {
    const int b = p.a[e], len = lane == 0 ? atomicExch(p.seq_lens + b, 0) : 0;
    free_row(p, b, __shfl_sync(0xffffffffu, len, 0), lane, 32);
  }
}

// The first `rows` slots of page `from` to page `to`, the heads of part `part`, one layer's keys or values, by the block.
constexpr int kCopyThreads = 256;
template <typename V>
__device__ __forceinline__ void copy_page(const PagesParams &p, const CacheRef &c, int layer, int from, int to, int rows, int part) {
  const int h0 = part * p.part_heads, heads = min(p.part_heads, p.heads - h0);
  const char *src = c.ptr + layer * c.sl + from * c.sp + h0 * c.sh;
  char *dst = c.ptr + layer * c.sl + to * c.sp + h0 * c.sh;
  const bool dense = c.st == p.row_bytes;                   // a head's rows lie one behind the other
  const bool whole = dense && rows == p.page_size && c.sh == (long long)p.row_bytes * p.page_size;      // and so do its heads
  const int per_head = rows * p.per_row, work = heads * per_head;
  constexpr int kDeep = 4;
  // a division for the head, where its copies are not one run with the next one's: by the block's own number of rows
  const float per = 1.0f / (float)per_head;
  for (int e0 = threadIdx.x; e0 < work; e0 += kDeep * kCopyThreads) {
    V x[kDeep];
    long long at[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int e = e0 + i * kCopyThreads;
      at[i] = -1;
      if (e < work) {
        if (whole) {
          at[i] = (long long)e * (int)sizeof(V);
        } else {
          int h = min((int)((float)e * per), heads - 1), in = e - h * per_head;      // off by one at most
          if (in < 0) { --h; in += per_head; }
          if (in >= per_head) { ++h; in -= per_head; }
          if (dense) {
            at[i] = h * c.sh + in * (int)sizeof(V);
          } else {
            const int r = p.by_row.of(in);
            at[i] = h * c.sh + r * c.st + (in - r * p.per_row) * (int)sizeof(V);
          }
        }
        x[i] = *reinterpret_cast<const V *>(src + at[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (at[i] >= 0) *reinterpret_cast<V *>(dst + at[i]) = x[i];
  }
}

// header of `work`: [0] fork: whether there is something to carry out, [1] compact: pages to move, [2] live pages
// fork: behind the lists, for each pair the source's length and the page that its copied rows get (or -1)
__device__ __forceinline__ int *fork_plan(const PagesParams &p) { return p.work + kPagesHeader + 2 * p.num_pages + p.max_seqs; }

// Whether the rows of a fork's sources name pages.  Looked at before anything is given out: a destination whose last page could
// not be filled would hold what that page's last owner left there.  A warp takes eight rows at a time, whose loads are on their
// way together, and where rows are few each is cut into 2^shift parts.  (64 forks of 5 to 27 pages, extended and freed: 29.1 us with
// eight rows, 29.4 with four, 32.6 with one; 4 forks of 8192 pages: 29.7 us, 142 with whole rows.)
__device__ __forceinline__ bool source_rows_ok(const PagesParams &p) {
  constexpr int kRows = 8;
  const int lane = threadIdx.x & 31, at_once = (int)(blockDim.x >> 5) * kRows;
  const int shift = max(__clz(p.n - 1) - 1 - __clz(at_once), 0), total = p.n << shift;
  bool ok = true;
  for (int q0 = (threadIdx.x >> 5) * kRows; q0 < total; q0 += at_once) {
    const int q = q0 + lane;
    int s = 0, begin = 0, count = 0;
    if (lane < kRows && q < total) {
      s = p.a[q >> shift];
      const int pages = pages_for(p, p.seq_lens[s]), span = (((pages + (1 << shift) - 1) >> shift) + 31) & ~31;
      begin = (q & ((1 << shift) - 1)) * span;
      count = min(pages - begin, span);
    }
    const int most = __reduce_max_sync(0xffffffffu, count);
    for (int j0 = 0; j0 < most; j0 += 32) {
      int page[kRows];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const long long at = __shfl_sync(0xffffffffu, s, k) * p.table_stride + __shfl_sync(0xffffffffu, begin, k) + j0 + lane;
        page[k] = j0 + lane < __shfl_sync(0xffffffffu, count, k) ? p.page_table[at] : 0;
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int seq = __shfl_sync(0xffffffffu, s, k);
        if ((unsigned)page[k] >= (unsigned)p.num_pages) {
          ok = false;
          report(p.status, SB_DEV_BAD_PAGE, seq);
        }
      }
    }
  }
  return ok;
}

__global__ void __launch_bounds__(kBookThreads) fork_plan_kernel(const __grid_constant__ PagesParams p) {
  __shared__ Book book;
  int *const shared = book.scan;
  enter_kernel<true>();
  int *list = p.work + kPagesHeader, *const mark = p.max_seqs <= kShort ? book.other : list + 2 * p.num_pages, *const plan = fork_plan(p);
  if (threadIdx.x == 0) p.work[0] = 0;
  for (int i = threadIdx.x; i < p.max_seqs; i += blockDim.x) mark[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
    const int s = p.a[i], d = p.b[i];
    int wrong = -1;
    if ((unsigned)s >= (unsigned)p.max_seqs) wrong = s;
    else if ((unsigned)d >= (unsigned)p.max_seqs || p.seq_lens[d] != 0 || atomicExch(mark + d, 1) != 0) wrong = d;
    else if (!length_ok(p, p.seq_lens[s])) wrong = s;
    else continue;
    bad = true;
    report(p.status, SB_DEV_BAD_SEQUENCE, wrong);
  }
  if (__syncthreads_or(bad)) return;
  for (int i = threadIdx.x; i < p.n; i += blockDim.x)
    if (mark[p.a[i]] != 0) {                  // a sequence cannot be forked and be a fork in one call
      bad = true;
      report(p.status, SB_DEV_BAD_SEQUENCE, p.a[i]);
    }
  bad |= !source_rows_ok(p);
  if (__syncthreads_or(bad)) return;
  int want = 0;
  for (int base = 0; base < p.n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int len = 0;
    if (i < p.n) len = p.seq_lens[p.a[i]];
    const int need = len % p.page_size != 0;
    int all;
    const int rank = want + block_scan(need, shared, all);
    if (i < p.n) {
      plan[2 * i] = len;
      plan[2 * i + 1] = need ? rank : -1;
    }
    want += all;
  }
  if (want <= kShort) list = book.list;
  if (want > p.num_pages || !list_free(p, want, list, shared)) {
    if (threadIdx.x == 0) report(p.status, SB_DEV_OUT_OF_PAGES, want);
    return;
  }
  for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
    const int rank = plan[2 * i + 1];
    if (rank >= 0) {
      plan[2 * i + 1] = list[rank];
      p.refs[list[rank]] = 1;
    }
    p.seq_lens[p.b[i]] = plan[2 * i];
  }
  if (threadIdx.x == 0) p.work[0] = 1;
}

// Blocks (part, pair): the parts of a pair are shares of its layers' keys and values, and first its row of the table, whose pages
// the plan has looked at.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) fork_kernel(const __grid_constant__ PagesParams p) {
  enter_kernel<true>();
  if (p.work[0] == 0) return;
  const int pair = blockIdx.y, part = blockIdx.x;
  const int *plan = fork_plan(p);
  const int len = plan[2 * pair], fresh = plan[2 * pair + 1], full = len / p.page_size, rest = len - full * p.page_size;
  const int *from = p.page_table + p.a[pair] * p.table_stride;
  int *to = p.page_table + p.b[pair] * p.table_stride;
  if (part == 0) {
    for (int i = threadIdx.x; i < full; i += kCopyThreads) {
      const int page = from[i];
      atomicAdd(p.refs + page, 1);
      to[i] = page;
    }
    if (threadIdx.x == 0 && rest > 0) to[full] = fresh;
    return;
  }
  if (rest == 0) return;
  const int job = p.by_parts.of(part - 1);
  copy_page<V>(p, job & 1 ? p.v : p.k, job >> 1, from[full], fresh, rest, part - 1 - job * p.parts);
}

__global__ void __launch_bounds__(kBookThreads) compact_plan_kernel(const __grid_constant__ PagesParams p) {
  __shared__ int shared[33];
  enter_kernel<true>();
  int *pairs = p.work + kPagesHeader, *place = pairs + p.num_pages;    // (hole, page) pairs, no more than half the pages; which pair a page is in
  int live = 0, mine = 0, negative = -1;
  bool bad = false;
  for (int b = threadIdx.x; b < p.max_seqs; b += blockDim.x)
    if (!length_ok(p, p.seq_lens[b])) {      // which entries of its row are to follow their pages, nothing says
      bad = true;
      report(p.status, SB_DEV_BAD_SEQ_LEN, b);
    }
  for (int base = 0; base < p.num_pages; base += (int)blockDim.x * kPer) {
    const int first = base + threadIdx.x * kPer;
    int x[kPer];
    read_refs(p, first, x);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      mine += x[i] > 0;
      if (x[i] < 0 && first + i < p.num_pages) negative = first + i;
    }
  }
  if (negative >= 0) report(p.status, SB_DEV_BAD_COUNT, negative);      // neither free nor in use: there would be fewer holes than pages to move
  if (__syncthreads_or(bad || negative >= 0)) {
    if (threadIdx.x == 0) p.work[1] = 0;
    return;
  }
  block_scan(mine, shared, live);
  int holes = 0, moved = 0;
  for (int base = 0; base < p.num_pages; base += (int)blockDim.x * kPer) {
    const int first = base + threadIdx.x * kPer;
    int x[kPer], h = 0, m = 0, all_h, all_m;
    read_refs(p, first, x);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      h += first + i < live && x[i] == 0;
      m += first + i >= live && x[i] > 0;
    }
    int rank_h = holes + block_scan(h, shared, all_h), rank_m = moved + block_scan(m, shared, all_m);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (first + i < live && x[i] == 0) pairs[2 * rank_h++] = first + i;
      if (first + i >= live && x[i] > 0) pairs[2 * rank_m++ + 1] = first + i;
    }
    holes += all_h;
    moved += all_m;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < moved; r += blockDim.x) {
    const int to = pairs[2 * r], from = pairs[2 * r + 1];
    place[from] = r;
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    p.work[1] = moved;
    p.work[2] = live;
  }
}

// Blocks below copy_blocks copy the moved pages, a share of a (page, layer, keys or values) at a time; the others rewrite the tables.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) compact_kernel(const __grid_constant__ PagesParams p, int copy_blocks) {
  enter_kernel<true>();
  const int moved = p.work[1], live = p.work[2];
  const int *pairs = p.work + kPagesHeader, *place = pairs + p.num_pages;
  if ((int)blockIdx.x < copy_blocks) {
    const int per_pair = p.layers * 2 * p.parts;
    const long long jobs = (long long)moved * per_pair;
    for (long long j = blockIdx.x; j < jobs; j += copy_blocks) {
      const int r = (int)(j / per_pair), in = (int)(j - (long long)r * per_pair), job = p.by_parts.of(in);
      copy_page<V>(p, job & 1 ? p.v : p.k, job >> 1, pairs[2 * r + 1], pairs[2 * r], p.page_size, in - job * p.parts);
    }
    return;
  }
  if (moved == 0) return;
  for (int b = blockIdx.x - copy_blocks; b < p.max_seqs; b += gridDim.x - copy_blocks) {
    const int pages = pages_for(p, p.seq_lens[b]);
    int *row = p.page_table + b * p.table_stride;
    for (int i = threadIdx.x; i < pages; i += kCopyThreads) {
      const int page = row[i];
      if ((unsigned)page < (unsigned)live) continue;
      // no page, or a free one, in whose place there is anything: stays as it is
      const int pair = (unsigned)page < (unsigned)p.num_pages ? place[page] : -1;
      if ((unsigned)pair < (unsigned)moved && pairs[2 * pair + 1] == page) row[i] = pairs[2 * pair];
      else report(p.status, SB_DEV_BAD_PAGE, b);
    }
  }
}

}  // namespace

cudaError_t launch_append(const AppendParams &p, cudaStream_t s) {
  const long long all = p.cu != nullptr ? p.tokens : p.tokens * p.num_seq;
  AppendParams q = p;
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  // A block's lookups are three trips to memory before its first copy: blocks enough that others' copies are under way meanwhile.
  // (34006 tokens x 8 heads x 128, bf16: 51, 49, 47, 55 us with 8, 16, 32, 64 blocks per SM.)
  q.per_block = (int)std::min<long long>(kMaxTokens, std::max<long long>(1, all / (kAppendBlocks * sms)));
  const dim3 grid((unsigned)((all + q.per_block - 1) / q.per_block));
  auto go = [&](auto kernel, int unit) {
    q.per_row = p.head_dim * p.esize / unit;
    q.per_token = 2 * p.kv_heads * q.per_row;
    q.by_row = FastDiv::by(q.per_row);
    q.by_token = FastDiv::by(q.per_token);
    return launch_kernel(kernel, grid, kAppendThreads, 0, s, q);
  };
  auto aligned = [&](const char *ptr, std::initializer_list<long long> strides) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return false;
    for (long long x : strides)
      if (x * p.esize % 16 != 0) return false;
    return true;
  };
  if (p.head_dim * p.esize % 16 == 0 && aligned(p.k.ptr, {p.k.sb, p.k.sh, p.k.st}) && aligned(p.v.ptr, {p.v.sb, p.v.sh, p.v.st}) &&
      aligned(p.kc.ptr, {p.kc.sp, p.kc.sh, p.kc.st}) && aligned(p.vc.ptr, {p.vc.sp, p.vc.sh, p.vc.st}))
    return go(append_kernel<uint4>, 16);
  if (p.esize == 4) return go(append_kernel<uint32_t>, 4);
  return go(append_kernel<unsigned short>, 2);
}

cudaError_t launch_extend(const PagesParams &p, cudaStream_t s) { return launch_kernel(extend_kernel, dim3(1), book_threads(p), 0, s, p); }

cudaError_t launch_free(const PagesParams &p, cudaStream_t s) {
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  return launch_kernel(free_kernel, dim3(std::min(p.n, kFreeBlocks * sms)), kFreeThreads, 0, s, p);
}

// A page's heads are shared out so that there are `blocks` pieces of work, or each is one head's.
static void set_parts(PagesParams &p, long long jobs, long long blocks) {
  const long long parts = std::min<long long>(p.heads, std::max<long long>(1, (blocks + jobs - 1) / jobs));
  p.part_heads = (int)((p.heads + parts - 1) / parts);
  p.parts = (p.heads + p.part_heads - 1) / p.part_heads;
  p.per_row = p.row_bytes / p.vec;
  p.by_row = FastDiv::by(p.per_row);
  p.by_parts = FastDiv::by(p.parts);
}

cudaError_t launch_fork(const PagesParams &params, cudaStream_t s, int *launches) {
  PagesParams p = params;
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  if ((e = launch_kernel(fork_plan_kernel, dim3(1), book_threads(p), 0, s, p)) != cudaSuccess) return e;
  *launches += 2;
  set_parts(p, 2LL * p.layers * p.n, 16LL * sms);
  const dim3 grid(1 + 2 * p.layers * p.parts, p.n);
  switch (p.vec) {
    case 16: return launch_kernel(fork_kernel<uint4>, grid, kCopyThreads, 0, s, p);
    case 4: return launch_kernel(fork_kernel<uint32_t>, grid, kCopyThreads, 0, s, p);
    default: return launch_kernel(fork_kernel<unsigned short>, grid, kCopyThreads, 0, s, p);
  }
}

cudaError_t launch_compact(const PagesParams &params, cudaStream_t s, int *launches) {
  PagesParams p = params;
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  if ((e = launch_kernel(compact_plan_kernel, dim3(1), book_threads(p), 0, s, p)) != cudaSuccess) return e;
  *launches += 2;
  set_parts(p, 1, p.heads);      // how many pages will move only the device knows: a head at a time
  const int copy_blocks = 8 * sms, table_blocks = std::min(p.max_seqs, sms);
  const dim3 grid(copy_blocks + table_blocks);
  switch (p.vec) {
    case 16: return launch_kernel(compact_kernel<uint4>, grid, kCopyThreads, 0, s, p, copy_blocks);
    case 4: return launch_kernel(compact_kernel<uint32_t>, grid, kCopyThreads, 0, s, p, copy_blocks);
    default: return launch_kernel(compact_kernel<unsigned short>, grid, kCopyThreads, 0, s, p, copy_blocks);
  }
}

}  // namespace sb
