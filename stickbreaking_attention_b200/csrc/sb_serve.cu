// C entry points of the serving operators: argument checks, workspace layout, kernel selection.
#include <algorithm>
#include <cstring>

#include "sb_decode.cuh"
#include "sb_pages.cuh"

namespace sb {

namespace {

constexpr int kMostPages = 1 << 20;      // of the keeping operators: the deciding block reads the counts of all of them

int esize_of(int dtype) { return dtype == SB_DTYPE_F32 ? 4 : 2; }

int check_strides(const char *name, const int64_t *stride, const int64_t *extent, int n, bool written) {
  for (int i = 0; i < n; ++i) {
    if (stride[i] < 0) return fail(SB_ERR_ARGUMENT, "%s has a negative stride", name);
    if (written && stride[i] == 0 && extent[i] > 1) return fail(SB_ERR_ARGUMENT, "%s repeats its elements and cannot be written to", name);
  }
  return SB_OK;
}
int check_cache(const char *name, const SbCache &c, int layers, int pages, int heads, int slots, bool written) {
  if (c.ptr == nullptr) return fail(SB_ERR_ARGUMENT, "%s.ptr is NULL", name);
  const int64_t stride[] = {c.stride_layer, c.stride_page, c.stride_h, c.stride_t}, extent[] = {layers, pages, heads, slots};
  return check_strides(name, stride, extent, 4, written);
}
int check_pool(int dtype, int kv_heads, int head_dim, int page_size, int num_pages, int max_pages) {
  if (dtype < SB_DTYPE_F32 || dtype > SB_DTYPE_F16) return fail(SB_ERR_ARGUMENT, "unknown dtype %d", dtype);
  if (kv_heads < 1 || kv_heads > 16384) return fail(SB_ERR_ARGUMENT, "kv_heads %d outside 1..16384", kv_heads);
  if (head_dim < 1 || head_dim > 256) return fail(SB_ERR_ARGUMENT, "head_dim %d outside 1..256", head_dim);
  if (page_size < 1 || page_size > 65536) return fail(SB_ERR_ARGUMENT, "page_size %d outside 1..65536", page_size);
  if (num_pages < 1) return fail(SB_ERR_ARGUMENT, "num_pages must be >= 1");
  if (max_pages < 1) return fail(SB_ERR_ARGUMENT, "max_pages must be >= 1");
  return SB_OK;
}

struct DecodePlan {
  int path, rows, rows_per_block, row_blocks, chunks, unit_shift, part_cols;
  bool by_item;
  size_t part_o, part_l, bytes;
};

int check_decode(const SbDecodeParams *p) {
  if (p == nullptr) return fail(SB_ERR_ARGUMENT, "params is NULL");
  if (p->struct_bytes != (int)sizeof(SbDecodeParams))
    return fail(SB_ERR_ARGUMENT, "struct_bytes %d != sizeof(SbDecodeParams) %d", p->struct_bytes, (int)sizeof(SbDecodeParams));
  if (p->reserved != 0) return fail(SB_ERR_ARGUMENT, "reserved must be 0");
  int rc = check_pool(p->dtype, p->kv_heads, p->head_dim, p->page_size, p->num_pages, p->max_pages);
  if (rc) return rc;
  if (p->batch < 0 || p->batch > (1 << 20)) return fail(SB_ERR_ARGUMENT, "batch outside 0..2^20");
  if (p->heads < 1 || p->heads > 65535 || p->heads % p->kv_heads != 0)
    return fail(SB_ERR_ARGUMENT, "heads %d must be a multiple of kv_heads %d (and at most 65535)", p->heads, p->kv_heads);
  if (p->new_tokens < 1 || p->new_tokens > 1024) return fail(SB_ERR_ARGUMENT, "new_tokens %d outside 1..1024", p->new_tokens);
  return SB_OK;
}

int plan_decode(const SbDecodeParams *p, DecodePlan &pl) {
  // whole 16-byte chunks in every row of the cache and no axis that repeats its elements, pairs of elements in q
  auto chunks = [p](const SbCache &c) {
    auto axis = [](int extent, int64_t stride) { return extent <= 1 || (stride > 0 && stride % 8 == 0); };
    return reinterpret_cast<uintptr_t>(c.ptr) % 16 == 0 && axis(p->num_pages, c.stride_page) && axis(p->kv_heads, c.stride_h) &&
           axis(p->page_size, c.stride_t);
  };
  const bool q_pairs = reinterpret_cast<uintptr_t>(p->q.ptr) % 4 == 0 && p->q.stride_b % 2 == 0 && p->q.stride_h % 2 == 0 && p->q.stride_t % 2 == 0;
  const bool tc = q_pairs && p->dtype != SB_DTYPE_F32 && !(p->flags & SB_FLAG_FORCE_SIMT) && p->head_dim % 8 == 0 && chunks(p->k) && chunks(p->v);
  pl.path = tc ? SB_PATH_TCGEN05 : SB_PATH_SIMT;
  pl.rows = p->heads / p->kv_heads * p->new_tokens;
  pl.rows_per_block = tc ? decode_tc_rows(pl.rows, p->head_dim) : decode_simt_rows(pl.rows, p->head_dim);
  pl.row_blocks = (pl.rows + pl.rows_per_block - 1) / pl.rows_per_block;
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return fail(SB_ERR_CUDA, "SM count: %s", cudaGetErrorString(e));
  pl.chunks = sms * (tc ? decode_tc_warps(pl.rows_per_block, p->head_dim) : decode_simt_warps(pl.rows_per_block, p->head_dim));
  const long long items = (long long)p->batch * p->kv_heads * pl.row_blocks;
  pl.by_item = items < pl.chunks;
  pl.part_cols = tc ? decode_tc_cols(p->head_dim) : p->head_dim;
  if (items > (1LL << 30)) return fail(SB_ERR_ARGUMENT, "batch * kv_heads too large");
  const long long longest = std::min<long long>((long long)p->max_pages * p->page_size, kMostTokens);
  pl.unit_shift = 4;                         // the units of all items have to be counted in 31 bits
  while (items * ((longest >> pl.unit_shift) + 1) > 0x7fffffffLL) ++pl.unit_shift;
  const size_t slots = 2 * (size_t)pl.chunks * pl.rows_per_block, notes = (size_t)(pl.by_item ? items : pl.chunks) * sizeof(int4);
  pl.part_o = (notes + 255) / 256 * 256;
  pl.part_l = pl.part_o + (slots * pl.part_cols + 128) * sizeof(float);      // (padded: see launch_decode_join)
  pl.bytes = (pl.part_l + slots * sizeof(float) + 255) / 256 * 256;
  return SB_OK;
}

TensorRef ref_of(const SbTensor &t) {
  return TensorRef{reinterpret_cast<char *>(t.ptr), (long long)t.stride_b, (long long)t.stride_h, (long long)t.stride_t};
}
PagedRef paged(const SbCache &c) {
  return PagedRef{reinterpret_cast<const char *>(c.ptr), (long long)c.stride_page, (long long)c.stride_h, (long long)c.stride_t};
}
CacheRef cache(const SbCache &c, long long unit) {
  return CacheRef{reinterpret_cast<char *>(c.ptr), c.stride_layer * unit, c.stride_page * unit, c.stride_h * unit, c.stride_t * unit};
}
int check_workspace(const void *ptr, size_t bytes, size_t need) {
  if (ptr == nullptr || bytes < need) return fail(SB_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", bytes, need);
  if (reinterpret_cast<uintptr_t>(ptr) % 256) return fail(SB_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  return SB_OK;
}

int run_decode(const SbDecodeParams *p, void *stream) {
  int *launches = begin_call();
  DecodePlan pl;
  int rc = check_decode(p);
  if (rc) return rc;
  if (p->batch == 0) return SB_OK;
  if (p->q.ptr == nullptr || p->o.ptr == nullptr || p->rem == nullptr || p->page_table == nullptr || p->seq_lens == nullptr)
    return fail(SB_ERR_ARGUMENT, "q, o, rem, page_table or seq_lens is NULL");
  const int64_t qs[] = {p->q.stride_b, p->q.stride_h, p->q.stride_t}, os[] = {p->o.stride_b, p->o.stride_h, p->o.stride_t};
  const int64_t extent[] = {p->batch, p->heads, p->new_tokens};
  if ((rc = check_strides("q", qs, extent, 3, false)) || (rc = check_strides("o", os, extent, 3, true)) ||
      (rc = check_cache("k", p->k, 1, p->num_pages, p->kv_heads, p->page_size, false)) ||
      (rc = check_cache("v", p->v, 1, p->num_pages, p->kv_heads, p->page_size, false)) ||
      (rc = device_ok()) || (rc = plan_decode(p, pl)) || (rc = check_workspace(p->workspace, p->workspace_bytes, pl.bytes)))
    return rc;
  DecodeParams k;
  memset(&k, 0, sizeof(k));
  k.q = ref_of(p->q);
  k.o = ref_of(p->o);
  k.rem = reinterpret_cast<char *>(p->rem);
  k.k = paged(p->k);
  k.v = paged(p->v);
  k.page_table = p->page_table;
  k.table_stride = p->page_table_stride;
  k.seq_lens = p->seq_lens;
  k.batch = p->batch; k.heads = p->heads; k.kv_heads = p->kv_heads; k.new_tokens = p->new_tokens; k.head_dim = p->head_dim;
  k.page_size = p->page_size; k.num_pages = p->num_pages; k.max_pages = p->max_pages;
  k.rows = pl.rows; k.row_blocks = pl.row_blocks; k.rows_per_block = pl.rows_per_block;
  k.attend_current = p->attend_current ? 1 : 0;
  k.dense = (p->flags & SB_FLAG_DENSE_ROW_PASS) ? 1 : 0;
  k.scale = p->logit_scale;
  k.chunks = pl.chunks;
  k.by_item = pl.by_item;
  k.part_cols = pl.part_cols;
  k.unit_shift = pl.unit_shift;
  k.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p->page_size == 1 << i) k.page_shift = i;
  // keys have 31 bits, so with 2^l >= page_size > 2^(l - 1) the quotient is exactly key * ceil(2^(31 + l) / page_size) >> 31 + l
  int l = 0;
  while ((1LL << l) < p->page_size) ++l;
  k.page_magic = (unsigned)(((1ULL << (31 + l)) + p->page_size - 1) / p->page_size);
  k.page_post = l - 1;
  k.items_per_seq = p->kv_heads * pl.row_blocks;
  char *ws = reinterpret_cast<char *>(p->workspace);
  k.notes = reinterpret_cast<int4 *>(ws);
  k.part_o = reinterpret_cast<float *>(ws + pl.part_o);
  k.part_l = reinterpret_cast<float *>(ws + pl.part_l);
  k.status = p->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = pl.path == SB_PATH_SIMT ? launch_decode_simt(k, p->dtype, s) : launch_decode_tc(k, p->dtype, s);
  if (e == cudaSuccess) e = pl.path == SB_PATH_SIMT ? launch_decode_join(k, p->dtype, s) : launch_decode_tc_join(k, p->dtype, s);
  *launches = 2;
  return e == cudaSuccess ? SB_OK : fail(SB_ERR_CUDA, "decode launch: %s", cudaGetErrorString(e));
}

int run_append(const SbAppendParams *p, void *stream) {
  int *launches = begin_call();
  int rc;
  if (p == nullptr) return fail(SB_ERR_ARGUMENT, "params is NULL");
  if (p->struct_bytes != (int)sizeof(SbAppendParams))
    return fail(SB_ERR_ARGUMENT, "struct_bytes %d != sizeof(SbAppendParams) %d", p->struct_bytes, (int)sizeof(SbAppendParams));
  if ((rc = check_pool(p->dtype, p->kv_heads, p->head_dim, p->page_size, p->num_pages, p->max_pages))) return rc;
  if (p->num_seq < 0 || p->num_seq > (1 << 20)) return fail(SB_ERR_ARGUMENT, "num_seq outside 0..2^20");
  if (p->tokens < 0 || p->tokens > 0x7fffff00LL || (p->cu_seqlens == nullptr && p->tokens * p->num_seq > 0x7fffff00LL))
    return fail(SB_ERR_ARGUMENT, "tokens out of range");
  if (p->num_seq == 0 || p->tokens == 0) return SB_OK;
  if (p->k.ptr == nullptr || p->v.ptr == nullptr || p->page_table == nullptr || p->seq_lens == nullptr)
    return fail(SB_ERR_ARGUMENT, "k, v, page_table or seq_lens is NULL");
  const int64_t ks[] = {p->k.stride_b, p->k.stride_h, p->k.stride_t}, vs[] = {p->v.stride_b, p->v.stride_h, p->v.stride_t};
  const int64_t extent[] = {1, 1, 1};
  if ((rc = check_strides("k", ks, extent, 3, false)) || (rc = check_strides("v", vs, extent, 3, false)) ||
      (rc = check_cache("k_cache", p->k_cache, 1, p->num_pages, p->kv_heads, p->page_size, true)) ||
      (rc = check_cache("v_cache", p->v_cache, 1, p->num_pages, p->kv_heads, p->page_size, true)) || (rc = device_ok()))
    return rc;
  AppendParams k;
  memset(&k, 0, sizeof(k));
  k.k = ref_of(p->k);
  k.v = ref_of(p->v);
  k.kc = cache(p->k_cache, 1);
  k.vc = cache(p->v_cache, 1);
  k.page_table = p->page_table;
  k.table_stride = p->page_table_stride;
  k.seq_lens = p->seq_lens;
  k.cu = p->cu_seqlens;
  k.cu64 = p->cu_seqlens_int64;
  k.check_leading_zero = p->cu_seqlens != nullptr && (p->flags & SB_FLAG_CHECK_LEADING_ZERO);
  k.num_seq = p->num_seq; k.kv_heads = p->kv_heads; k.head_dim = p->head_dim; k.page_size = p->page_size;
  k.num_pages = p->num_pages; k.max_pages = p->max_pages; k.esize = esize_of(p->dtype);
  k.tokens = p->tokens;
  k.status = p->status;
  const cudaError_t e = launch_append(k, reinterpret_cast<cudaStream_t>(stream));
  *launches = 1;
  return e == cudaSuccess ? SB_OK : fail(SB_ERR_CUDA, "append launch: %s", cudaGetErrorString(e));
}

enum class Keep { kExtend, kFork, kFree, kCompact };

int check_pages(const SbPagesParams *p) {
  if (p == nullptr) return fail(SB_ERR_ARGUMENT, "params is NULL");
  if (p->struct_bytes != (int)sizeof(SbPagesParams))
    return fail(SB_ERR_ARGUMENT, "struct_bytes %d != sizeof(SbPagesParams) %d", p->struct_bytes, (int)sizeof(SbPagesParams));
  if (p->reserved != 0) return fail(SB_ERR_ARGUMENT, "reserved must be 0");
  if (p->max_seqs < 1 || p->max_seqs > (1 << 20)) return fail(SB_ERR_ARGUMENT, "max_seqs outside 1..2^20");
  if (p->max_pages < 1) return fail(SB_ERR_ARGUMENT, "max_pages must be >= 1");
  if (p->num_pages < 1 || p->num_pages > kMostPages) return fail(SB_ERR_ARGUMENT, "num_pages outside 1..2^20");
  if (p->page_size < 1 || p->page_size > 65536) return fail(SB_ERR_ARGUMENT, "page_size %d outside 1..65536", p->page_size);
  if (p->n < 0 || p->n > 65535) return fail(SB_ERR_ARGUMENT, "%d listed sequences: at most 65535", p->n);
  return SB_OK;
}
size_t pages_bytes(const SbPagesParams *p) {
  return ((size_t)pages_work_ints(p->num_pages, p->max_seqs, p->n) * sizeof(int) + 255) / 256 * 256;
}

int run_pages(const SbPagesParams *p, Keep what, void *stream) {
  int *launches = begin_call();
  int rc = check_pages(p);
  if (rc) return rc;
  if (p->page_table == nullptr || p->seq_lens == nullptr || p->page_refs == nullptr)
    return fail(SB_ERR_ARGUMENT, "page_table, seq_lens or page_refs is NULL");
  if (p->max_seqs > 1 && p->page_table_stride < p->max_pages) return fail(SB_ERR_ARGUMENT, "the rows of page_table overlap");
  if ((what == Keep::kFork || what == Keep::kFree) && p->n == 0) return SB_OK;
  if ((what == Keep::kFork && (p->first == nullptr || p->second == nullptr)) || (what == Keep::kFree && p->first == nullptr))
    return fail(SB_ERR_ARGUMENT, "the listed sequences are missing");
  if (what == Keep::kExtend && p->first == nullptr && p->count < 0) return fail(SB_ERR_ARGUMENT, "count is negative");
  if (what != Keep::kFree && (rc = check_workspace(p->workspace, p->workspace_bytes, pages_bytes(p)))) return rc;
  PagesParams k;
  memset(&k, 0, sizeof(k));
  k.page_table = p->page_table;
  k.table_stride = p->page_table_stride;
  k.seq_lens = p->seq_lens;
  k.refs = p->page_refs;
  k.max_seqs = p->max_seqs; k.max_pages = p->max_pages; k.num_pages = p->num_pages; k.page_size = p->page_size;
  k.a = p->first;
  k.b = p->second;
  k.n = p->n;
  k.count = p->count;
  k.work = reinterpret_cast<int *>(p->workspace);
  k.status = p->status;
  if (what == Keep::kFork || what == Keep::kCompact) {
    if ((rc = check_pool(p->dtype, p->kv_heads, p->head_dim, p->page_size, p->num_pages, p->max_pages))) return rc;
    if (p->layers < 1 || p->layers > 65535) return fail(SB_ERR_ARGUMENT, "layers outside 1..65535");
    if ((rc = check_cache("k_cache", p->k_cache, p->layers, p->num_pages, p->kv_heads, p->page_size, true)) ||
        (rc = check_cache("v_cache", p->v_cache, p->layers, p->num_pages, p->kv_heads, p->page_size, true)))
      return rc;
    const int esize = esize_of(p->dtype);
    if ((long long)p->kv_heads * p->page_size * p->head_dim > 0x3fffffffLL) return fail(SB_ERR_ARGUMENT, "a page of more than 2^30 elements");
    k.k = cache(p->k_cache, esize);
    k.v = cache(p->v_cache, esize);
    k.layers = p->layers;
    k.heads = p->kv_heads;
    k.row_bytes = p->head_dim * esize;
    auto aligned = [](const CacheRef &c) {
      return reinterpret_cast<uintptr_t>(c.ptr) % 16 == 0 && c.sl % 16 == 0 && c.sp % 16 == 0 && c.sh % 16 == 0 && c.st % 16 == 0;
    };
    k.vec = k.row_bytes % 16 == 0 && aligned(k.k) && aligned(k.v) ? 16 : esize;
  }
  if ((rc = device_ok())) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  switch (what) {
    case Keep::kExtend: e = launch_extend(k, s); *launches = 1; break;
    case Keep::kFree: e = launch_free(k, s); *launches = 1; break;
    case Keep::kFork: e = launch_fork(k, s, launches); break;
    case Keep::kCompact: e = launch_compact(k, s, launches); break;
  }
  return e == cudaSuccess ? SB_OK : fail(SB_ERR_CUDA, "page keeping launch: %s", cudaGetErrorString(e));
}

}  // namespace

}  // namespace sb

extern "C" {

size_t sb_attn_decode_workspace_bytes(const SbDecodeParams *p) {
  sb::DecodePlan pl;
  return sb::check_decode(p) || sb::plan_decode(p, pl) ? (size_t)-1 : pl.bytes;
}

int sb_attn_decode(const SbDecodeParams *p, void *stream) { return sb::run_decode(p, stream); }

int sb_attn_decode_path(const SbDecodeParams *p) {
  sb::DecodePlan pl;
  return sb::check_decode(p) || sb::plan_decode(p, pl) ? -1 : pl.path;
}

int sb_kv_append(const SbAppendParams *p, void *stream) { return sb::run_append(p, stream); }

size_t sb_kv_pages_workspace_bytes(const SbPagesParams *p) { return sb::check_pages(p) ? (size_t)-1 : sb::pages_bytes(p); }

int sb_kv_extend(const SbPagesParams *p, void *stream) { return sb::run_pages(p, sb::Keep::kExtend, stream); }
int sb_kv_fork(const SbPagesParams *p, void *stream) { return sb::run_pages(p, sb::Keep::kFork, stream); }
int sb_kv_free(const SbPagesParams *p, void *stream) { return sb::run_pages(p, sb::Keep::kFree, stream); }
int sb_kv_compact(const SbPagesParams *p, void *stream) { return sb::run_pages(p, sb::Keep::kCompact, stream); }

}  // extern "C"
