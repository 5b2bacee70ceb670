// Attention of new tokens over a paged key-value cache: the CUDA-core kernel (fp32, and 16-bit tensors whose rows cannot be
// copied 16 bytes at a time) and the join of split items.
#include <algorithm>

#include "sb_decode.cuh"

namespace sb {

namespace {

__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}

// kCols: columns a lane holds (32 kCols >= head_dim); kRows: query rows.  As many warps as registers and shared memory allow: a
// tile is a long chain (16 dots, a scan, 16 sums), other warps' tiles fill it, and their copies are in flight as well.
// (fp32, 8 heads x 128 columns, 20 sequences of 157 to 8150 tokens: 122, 92, 73 us with 4, 6, 12 warps of 3, 2, 1 stages; 64 columns 76, 60
// with 8, 12 warps of 3, 2; 128 columns and 4 rows 124, 107 with 8, 12 of 1, although 12 warps leave 168 registers, of which those rows need
// 8 to 15 more; 256 columns, 157 to 4000 tokens, 132, 98 with 4, 6 of 1.)
template <int kCols, int kRows> struct SimtShape {
  static constexpr int kWidth = 32 * kCols;                              // floats of a row in shared memory
  static constexpr int kWarps = kCols <= 2 ? 12 : kCols <= 4 ? (kRows <= 4 ? 12 : 8) : 6;
  static constexpr int kStage = 2 * kTileKeys * kWidth * 4;              // 16 keys, 16 values
  static constexpr int kStages = 192 * 1024 / (kWarps * kStage);
  static constexpr int kBytes = kWarps * kStages * kStage;               // 192 KiB
};

template <int kCols> __device__ __forceinline__ void load_cols(const float *src, float (&x)[kCols]) {
  if constexpr (kCols == 2) {
    const float2 a = *reinterpret_cast<const float2 *>(src);
    x[0] = a.x; x[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < kCols; i += 4) {
      const float4 a = *reinterpret_cast<const float4 *>(src + i * 32);   // a chunk of 128 columns after the other
      x[i] = a.x; x[i + 1] = a.y; x[i + 2] = a.z; x[i + 3] = a.w;
    }
  }
}
// The column that element i of a lane is.
template <int kCols> __device__ __forceinline__ int col_of(int lane, int i) {
  return kCols == 2 ? lane * 2 + i : (i / 4) * 128 + lane * 4 + i % 4;
}

// The CUDA-core engine.  kRows: query rows (1, 2, 4, 8); kVec: bytes of a copy (fp32: 16 or 4; 16-bit types: 0, converted on the
// way).  Lane l holds the scores of row 2 pair + (l & 1) at key l >> 1 of the tile: 16 keys and two rows fill a warp, and the scan
// over keys takes four shuffles.  `left`: natural log of the stick that remains.
template <typename T, int kCols, int kRows, int kVec> struct SimtEngine : SimtShape<kCols, kRows> {
  using S = SimtShape<kCols, kRows>;
  using S::kWidth;
  static constexpr int kPairs = (kRows + 1) / 2;
  float q[kRows][kCols], acc[kRows][kCols];
  LongSum left[kPairs];
  int limit[kPairs];

  __device__ static __forceinline__ void prefetch_rows(const DecodeParams &p, const Piece &w) { prefetch_q(p, w, sizeof(T)); }

  __device__ static __forceinline__ void copy_run(const DecodeParams &p, const Piece &w, int page, int slot, char *to) {
    copy(p, w, page, slot + (threadIdx.x & 15), to);
  }
  // Rows without a page, and columns behind head_dim, are zeros.
  __device__ static __forceinline__ void copy(const DecodeParams &p, const Piece &w, int page, int slot, char *to) {
    const int lane = threadIdx.x & 31;
    for (int j = 0; j < kTileKeys; ++j) {
      const int pg = __shfl_sync(0xffffffffu, page, j), sl = __shfl_sync(0xffffffffu, slot, j);
      const bool take = pg >= 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const PagedRef &t = kv ? p.v : p.k;
        const T *row = reinterpret_cast<const T *>(t.ptr) + (take ? pg * t.sp + w.head * t.sh + sl * t.st : 0);
        float *dst = reinterpret_cast<float *>(to) + (kv * kTileKeys + j) * kWidth;
        if constexpr (kVec == 0) {
          for (int c = lane; c < kWidth; c += 32) dst[c] = take && c < p.head_dim ? to_f32<T>(row[c]) : 0.0f;
        } else {
          for (int c = lane * (kVec / 4); c < kWidth; c += 8 * kVec) {
            const bool in = take && c < p.head_dim;
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(dst + c);
            if constexpr (kVec == 16) cp_async16(at, row + (in ? c : 0), in);
            else cp_async4(at, row + (in ? c : 0), in);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void start(const DecodeParams &p, const Piece &w) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const T *row = reinterpret_cast<const T *>(p.q.ptr) + row_offset(p, p.q, w.seq, w.head, w.row0 + min(r, w.rows - 1));
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int c = col_of<kCols>(lane, i);
        q[r][i] = c < p.head_dim ? to_f32<T>(row[c]) : 0.0f;
        acc[r][i] = 0.0f;
      }
    }
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr) {
      left[pr] = LongSum();
      limit[pr] = row_limit(p, w.keys, w.row0 + min(2 * pr + (lane & 1), w.rows - 1));
    }
  }

  __device__ __forceinline__ void tile(const DecodeParams &p, const Piece &w, const char *stage, int key0) {
    const int lane = threadIdx.x & 31;
    const float *ks = reinterpret_cast<const float *>(stage) + (kCols == 2 ? 2 : 4) * lane, *vs = ks + kTileKeys * kWidth;
    float a[kPairs];
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr) {
      constexpr int two = kRows > 1 ? 2 : 1;
      float z[2][kTileKeys];
#pragma unroll
      for (int j = 0; j < kTileKeys; ++j) {
        float k[kCols];
        load_cols<kCols>(ks + j * kWidth, k);
#pragma unroll
        for (int r = 0; r < two; ++r) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < kCols; ++i) s = fmaf(q[2 * pr + r][i], k[i], s);
          z[r][j] = s;
        }
        if (two == 1) z[1][j] = 0.0f;
      }
      // each step adds two lanes up and halves the keys a lane still holds: bits 4..1 of the lane become the key, bit 0 the row
#pragma unroll
      for (int half = 8; half >= 1; half >>= 1) {
        const bool up = lane & (2 * half);
#pragma unroll
        for (int r = 0; r < two; ++r)
#pragma unroll
          for (int j = 0; j < half; ++j) {
            const float keep = up ? z[r][j + half] : z[r][j], give = up ? z[r][j] : z[r][j + half];
            z[r][j] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * half);
          }
      }
      const bool odd = lane & 1;
      const float keep = odd ? z[1][0] : z[0][0], give = odd ? z[0][0] : z[1][0];
      const float x = (keep + __shfl_xor_sync(0xffffffffu, give, 1)) * p.scale;
      const bool in = key0 + (lane >> 1) < limit[pr];
      const float l1 = log1pf(expf(-fabsf(x)));
      const float broken = in ? -(fmaxf(x, 0.0f) + l1) : 0.0f;      // log(1 - beta)
      float sum = broken;                                            // over this and the tile's later keys
#pragma unroll
      for (int d = 2; d < 32; d <<= 1) {
        const float other = __shfl_down_sync(0xffffffffu, sum, d);
        if (lane + d < 32) sum += other;
      }
      float later = __shfl_down_sync(0xffffffffu, sum, 2);
      if (lane >= 30) later = 0.0f;
      a[pr] = in ? expf((fminf(x, 0.0f) - l1) + (left[pr].sum + later)) : 0.0f;
      left[pr].add(__shfl_sync(0xffffffffu, sum, lane & 1));
    }
    // a value that a row does not attend to is left out, not multiplied by 0: it may be no number
    const bool edge = key0 + kTileKeys > w.edge;
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      float v[kCols];
      load_cols<kCols>(vs + j * kWidth, v);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float weight = __shfl_sync(0xffffffffu, a[r / 2], 2 * j + (r & 1));
        if (edge && key0 + j >= __shfl_sync(0xffffffffu, limit[r / 2], r & 1)) continue;
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[r][i] = fmaf(weight, v[i], acc[r][i]);
      }
    }
  }

  __device__ __forceinline__ bool gone() const {
    bool all = true;
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr) all = all && left[pr].sum < kStickGone * (float)kLn2D;
    return __all_sync(0xffffffffu, all);
  }

  __device__ __forceinline__ void finish(const DecodeParams &p, const Piece &w, int slot, bool bad) {
    const int lane = threadIdx.x & 31;
    const float nan = __int_as_float(0x7fffffff);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= w.rows) break;
      const RowOut<T> out(p, w, slot, r);
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int c = col_of<kCols>(lane, i);
        if (c < p.head_dim) out.put(c, bad ? nan : acc[r][i]);
      }
    }
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr)
      if (lane < 2 && 2 * pr + lane < w.rows) put_rem<T>(p, w, slot, 2 * pr + lane, bad ? nan : left[pr].sum * kLog2e);
  }
};

template <typename E>
__global__ void __launch_bounds__(E::kWarps * 32, 1) decode_simt_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) char ring[];
  __shared__ ChunkShared<E::kWarps> shared;
  enter_kernel<true>();
  decode_chunks<E>(p, ring, shared);
}

// Joins the pieces of the items that were cut, up to 128 columns of one row at a time, newest piece first.  Each warp has such a
// part of its own (kTogether 1), or kTogether warps have the same one and take a run of its pieces each, whose sums are joined
// like pieces.  The sticks of 32 pieces are one scan over the lanes, which leaves a product and a sum per piece and column.
constexpr int kJoinCols = 128, kJoinDeep = 8;

// Eight pieces' columns in flight together.  (One statement: left to itself the compiler loads a few, adds them up, and only then
// loads the next, which is a trip to L2 each.)
__device__ __forceinline__ void load_eight(const float *const (&at)[8], float (&x)[8][4]) {
  asm volatile(
      "ld.global.f32 %0, [%32];\n\tld.global.f32 %1, [%32+128];\n\tld.global.f32 %2, [%32+256];\n\tld.global.f32 %3, [%32+384];\n\t"
      "ld.global.f32 %4, [%33];\n\tld.global.f32 %5, [%33+128];\n\tld.global.f32 %6, [%33+256];\n\tld.global.f32 %7, [%33+384];\n\t"
      "ld.global.f32 %8, [%34];\n\tld.global.f32 %9, [%34+128];\n\tld.global.f32 %10, [%34+256];\n\tld.global.f32 %11, [%34+384];\n\t"
      "ld.global.f32 %12, [%35];\n\tld.global.f32 %13, [%35+128];\n\tld.global.f32 %14, [%35+256];\n\tld.global.f32 %15, [%35+384];\n\t"
      "ld.global.f32 %16, [%36];\n\tld.global.f32 %17, [%36+128];\n\tld.global.f32 %18, [%36+256];\n\tld.global.f32 %19, [%36+384];\n\t"
      "ld.global.f32 %20, [%37];\n\tld.global.f32 %21, [%37+128];\n\tld.global.f32 %22, [%37+256];\n\tld.global.f32 %23, [%37+384];\n\t"
      "ld.global.f32 %24, [%38];\n\tld.global.f32 %25, [%38+128];\n\tld.global.f32 %26, [%38+256];\n\tld.global.f32 %27, [%38+384];\n\t"
      "ld.global.f32 %28, [%39];\n\tld.global.f32 %29, [%39+128];\n\tld.global.f32 %30, [%39+256];\n\tld.global.f32 %31, [%39+384];"
      : "=f"(x[0][0]), "=f"(x[0][1]), "=f"(x[0][2]), "=f"(x[0][3]), "=f"(x[1][0]), "=f"(x[1][1]), "=f"(x[1][2]), "=f"(x[1][3]),
        "=f"(x[2][0]), "=f"(x[2][1]), "=f"(x[2][2]), "=f"(x[2][3]), "=f"(x[3][0]), "=f"(x[3][1]), "=f"(x[3][2]), "=f"(x[3][3]),
        "=f"(x[4][0]), "=f"(x[4][1]), "=f"(x[4][2]), "=f"(x[4][3]), "=f"(x[5][0]), "=f"(x[5][1]), "=f"(x[5][2]), "=f"(x[5][3]),
        "=f"(x[6][0]), "=f"(x[6][1]), "=f"(x[6][2]), "=f"(x[6][3]), "=f"(x[7][0]), "=f"(x[7][1]), "=f"(x[7][2]), "=f"(x[7][3])
      : "l"(at[0]), "l"(at[1]), "l"(at[2]), "l"(at[3]), "l"(at[4]), "l"(at[5]), "l"(at[6]), "l"(at[7])
      : "memory");
}

template <typename T, int kWarps, int kTogether>
__global__ void __launch_bounds__(kWarps * 32) decode_join_kernel(const __grid_constant__ DecodeParams p) {
  enter_kernel<true>();
  const int4 note = p.notes[blockIdx.x];
  if (note.w == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / kTogether, member = warp % kTogether;
  const int head = p.row_blocks == 1 ? note.y : note.y / p.row_blocks, row0 = (note.y - head * p.row_blocks) * p.rows_per_block;
  const int rows = min(p.rows - row0, p.rows_per_block), segments = (p.head_dim + kJoinCols - 1) / kJoinCols;
  const int job = blockIdx.y * (kWarps / kTogether) + team, r = segments == 1 ? job : job >> 1, col0 = segments == 1 ? 0 : (job & 1) * kJoinCols;
  const bool real = r < rows;
  if (kTogether == 1 && !real) return;
  const int share = (note.w + kTogether - 1) / kTogether;
  const int begin = real ? min(member * share, note.w) : 0, end = real ? min(begin + share, note.w) : 0;
  // i-th piece from the newest on: the oldest is its chunk's last, the others are their chunk's first
  const auto slot_of = [&](int i) { return 2LL * (note.z + note.w - 1 - i) + (i == note.w - 1 ? 1 : 0); };
  const long long part = (long long)p.rows_per_block * p.head_dim;
  const float *const parts = p.part_o + r * p.head_dim + col0 + lane;
  float o[4] = {}, left = 0.0f;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int n = min(end - i0, 32);
    const float own = lane < n ? p.part_l[slot_of(i0 + lane) * p.rows_per_block + r] : 0.0f;
    float x[kJoinDeep][4];
    const float *at[kJoinDeep];
    float sum = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    float before = __shfl_up_sync(0xffffffffu, sum, 1);
    if (lane == 0) before = 0.0f;
    const float stick = lane < n ? exp2_all(left + before) : 0.0f;      // what is left of the stick at the piece's newest end
    left += __shfl_sync(0xffffffffu, sum, 31);
    for (int k0 = 0; k0 < n; k0 += kJoinDeep) {
#pragma unroll
      for (int k = 0; k < kJoinDeep; ++k) at[k] = parts + slot_of(min(i0 + k0 + k, end - 1)) * part;
      load_eight(at, x);
#pragma unroll
      for (int k = 0; k < kJoinDeep; ++k) {
        const float w = __shfl_sync(0xffffffffu, stick, (k0 + k) & 31);
        const bool in = k0 + k < n && w != 0.0f;                        // (0 times what is no number stays out)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += in ? w * x[k][j] : 0.0f;
      }
    }
  }
  if constexpr (kTogether > 1) {
    __shared__ float sums[kWarps][4][32], lefts[kWarps];
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][j][lane] = o[j];
    if (lane == 0) lefts[warp] = left;
    __syncthreads();
    if (member != 0 || !real) return;
    left = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = 0.0f;
#pragma unroll
    for (int n = 0; n < kTogether; ++n) {
      const float w = exp2_all(left);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += w != 0.0f ? w * sums[warp + n][j][lane] : 0.0f;
      left += lefts[warp + n];
    }
  }
  T *const out = reinterpret_cast<T *>(p.o.ptr) + row_offset(p, p.o, note.x, head, row0 + r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = col0 + lane + 32 * j;
    if (c < p.head_dim) out[c] = from_f32<T>(o[j]);
  }
  if (lane == 0 && col0 == 0) reinterpret_cast<T *>(p.rem)[rem_index(p, note.x, head, row0 + r)] = from_f32<T>(exp2f(left));
}

template <typename E> cudaError_t launch_engine(const DecodeParams &p, cudaStream_t s) {
  const auto kernel = decode_simt_kernel<E>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), E::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3(p.chunks / E::kWarps), E::kWarps * 32, E::kBytes, s, p);
}
template <typename T, int kCols, int kVec> cudaError_t launch_rows(const DecodeParams &p, cudaStream_t s) {
  switch (p.rows_per_block) {
    case 1: return launch_engine<SimtEngine<T, kCols, 1, kVec>>(p, s);
    case 2: return launch_engine<SimtEngine<T, kCols, 2, kVec>>(p, s);
    case 4: return launch_engine<SimtEngine<T, kCols, 4, kVec>>(p, s);
  }
  if constexpr (kCols <= 4) return launch_engine<SimtEngine<T, kCols, 8, kVec>>(p, s);
  return cudaErrorInvalidValue;
}
template <typename T, int kVec> cudaError_t launch_cols(const DecodeParams &p, cudaStream_t s) {
  if (p.head_dim <= 64) return launch_rows<T, 2, kVec>(p, s);
  if (p.head_dim <= 128) return launch_rows<T, 4, kVec>(p, s);
  return launch_rows<T, 8, kVec>(p, s);
}

}  // namespace

// (Four rows of a head_dim over 128 need 26 registers more than a thread has; twice as many rows would need twice the accumulators.)
int decode_simt_rows(int rows, int head_dim) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 || head_dim > 128 ? 4 : 8; }
int decode_simt_warps(int rows, int head_dim) {
  if (head_dim <= 64) return SimtShape<2, 1>::kWarps;
  if (head_dim <= 128) return rows <= 4 ? SimtShape<4, 4>::kWarps : SimtShape<4, 8>::kWarps;
  return SimtShape<8, 1>::kWarps;
}

cudaError_t launch_decode_simt(const DecodeParams &p, int dtype, cudaStream_t s) {
  auto aligned = [](const PagedRef &t) {
    return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && t.sp % 4 == 0 && t.sh % 4 == 0 && t.st % 4 == 0;
  };
  switch (dtype) {
    case SB_DTYPE_F32: return p.head_dim % 4 == 0 && aligned(p.k) && aligned(p.v) ? launch_cols<float, 16>(p, s) : launch_cols<float, 4>(p, s);
    case SB_DTYPE_BF16: return launch_cols<__nv_bfloat16, 0>(p, s);
    default: return launch_cols<__half, 0>(p, s);
  }
}

// The columns behind head_dim that a part reads (up to 127) lie in the next row, or behind the last one in the padding that the
// workspace has there.  1, 4, 8 or 32 warps share a part, by the chunks that there are for an item.  (The whole call in us with 1, 4, 8, 32,
// fp32, 64 columns.  1.7 chunks per item, 64 sequences x 16 heads, 1024 tokens: 148.7, 148.5, 149.9, 164; 3.8, 29 x 16: 74.9, 74.5, 73.5, 81;
// 4.4, 25 x 16: 67.6, 66.6, 66.4, 72; 15, 15 x 8: 31, 29, 28.8, 29.2; 17, 13 x 8: 26.4, 24, 24.1, 24.4; 222, 1 x 8, 16384 tokens: 74, 39, 33.9, 29.9;
// 296, 1 x 6: 79, 32, 28.5, 24.7.)
cudaError_t launch_decode_join(const DecodeParams &p, int dtype, cudaStream_t s) {
  const long long items = (long long)p.batch * p.items_per_seq;
  const int notes = (int)(p.by_item ? items : p.chunks);
  const int jobs = p.rows_per_block * ((p.head_dim + kJoinCols - 1) / kJoinCols);
  const int together = p.chunks < 4 * items ? 1 : p.chunks < 16 * items ? 4 : p.chunks < 256 * items ? 8 : 32;
  auto go = [&](auto kernel, int warps, int per_block) {
    return launch_kernel(kernel, dim3(notes, (jobs + per_block - 1) / per_block), warps * 32, 0, s, p);
  };
#define SB_JOIN(T)                                               \
  together == 32  ? go(decode_join_kernel<T, 32, 32>, 32, 1)     \
  : together == 8 ? go(decode_join_kernel<T, 8, 8>, 8, 1)        \
  : together == 4 ? go(decode_join_kernel<T, 4, 4>, 4, 1)        \
                  : go(decode_join_kernel<T, 4, 1>, 4, 4)
  switch (dtype) {
    case SB_DTYPE_F32: return SB_JOIN(float);
    case SB_DTYPE_BF16: return SB_JOIN(__nv_bfloat16);
    default: return SB_JOIN(__half);
  }
#undef SB_JOIN
}

}  // namespace sb
