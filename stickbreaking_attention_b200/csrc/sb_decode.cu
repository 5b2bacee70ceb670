// Attention of new tokens over a paged key-value cache: the CUDA-core kernel (fp32, and 16-bit tensors whose rows cannot be
// copied 16 bytes at a time) and the join of split items.
#include "sb_decode.cuh"

namespace sb {

namespace {

__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
constexpr int kTileKeys = 16, kStages = 3;

// kCols: columns a lane holds (32 kCols >= head_dim); kRows: query rows (1, 2, 4, 8).
template <int kCols> struct SimtShape {
  static constexpr int kWidth = 32 * kCols;                              // floats of a row in shared memory
  static constexpr int kWarps = kCols <= 2 ? 8 : kCols <= 4 ? 4 : 2;     // 24 KiB (2 columns) to 96 KiB of stages per warp
  static constexpr int kStage = 2 * kTileKeys * kWidth;                  // floats of a stage: 16 keys, 16 values
  static constexpr int kBytes = kWarps * kStages * kStage * 4;
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

// A warp's copies of 16 keys and values into one stage.  Rows that no query attends to, and columns behind head_dim, are zeros.
// Returns whether the page table had an entry that is no page.
template <typename T, int kCols>
__device__ __forceinline__ bool load_stage(const DecodeParams &p, const Piece &w, int key0, int key_end, float *stage, bool vec) {
  using S = SimtShape<kCols>;
  const int lane = threadIdx.x & 31;
  int page = -1, slot = 0;
  const int key = key0 + lane;
  const bool wanted = lane < kTileKeys && key < key_end;
  if (wanted) {
    const int index = key / p.page_size;
    slot = key - index * p.page_size;
    page = page_of(p, w.seq, index);
  }
  const bool bad = __any_sync(0xffffffffu, wanted && page < 0);
  for (int j = 0; j < kTileKeys; ++j) {
    const int pg = __shfl_sync(0xffffffffu, page, j), sl = __shfl_sync(0xffffffffu, slot, j);
    const bool take = pg >= 0;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const PagedRef &t = kv ? p.v : p.k;
      const T *row = reinterpret_cast<const T *>(t.ptr) + (take ? pg * t.sp + w.head * t.sh + sl * t.st : 0);
      float *dst = stage + (kv * kTileKeys + j) * S::kWidth;
      if constexpr (sizeof(T) == 4) {
        if (vec) {
          for (int c = lane * 4; c < S::kWidth; c += 128) {
            const bool in = take && c < p.head_dim;
            cp_async16((uint32_t)__cvta_generic_to_shared(dst + c), row + (in ? c : 0), in);
          }
        } else {
          for (int c = lane; c < S::kWidth; c += 32) {
            const bool in = take && c < p.head_dim;
            cp_async4((uint32_t)__cvta_generic_to_shared(dst + c), row + (in ? c : 0), in);
          }
        }
      } else {
        for (int c = lane; c < S::kWidth; c += 32) dst[c] = take && c < p.head_dim ? to_f32<T>(row[c]) : 0.0f;
      }
    }
  }
  return bad;
}

// One warp's keys, newest first, summed up in (acc, left): left = natural log of the stick that remains.  Lane l holds
// the scores of row 2 pair + (l & 1) at key l >> 1 of the tile: 16 keys and two rows fill a warp, and the scan over keys takes
// four shuffles.
template <typename T, int kCols, int kRows> struct SimtWarp {
  static constexpr int kPairs = (kRows + 1) / 2;
  float q[kRows][kCols], acc[kRows][kCols];
  double left[kPairs];
  int limit[kPairs];

  __device__ __forceinline__ void tile(const DecodeParams &p, const Piece &w, const float *stage, int key0) {
    using S = SimtShape<kCols>;
    const int lane = threadIdx.x & 31;
    const float *ks = stage + (kCols == 2 ? 2 : 4) * lane, *vs = ks + kTileKeys * S::kWidth;
    float a[kPairs];
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr) {
      constexpr int two = kRows > 1 ? 2 : 1;
      float z[2][kTileKeys];
#pragma unroll
      for (int j = 0; j < kTileKeys; ++j) {
        float k[kCols];
        load_cols<kCols>(ks + j * S::kWidth, k);
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
      a[pr] = in ? expf((fminf(x, 0.0f) - l1) + ((float)left[pr] + later)) : 0.0f;
      left[pr] += (double)__shfl_sync(0xffffffffu, sum, lane & 1);
    }
    // a value that a row does not attend to is left out, not multiplied by 0: it may be no number
    const bool edge = key0 + kTileKeys > w.edge;
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      float v[kCols];
      load_cols<kCols>(vs + j * S::kWidth, v);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float weight = __shfl_sync(0xffffffffu, a[r / 2], 2 * j + (r & 1));
        if (edge && key0 + j >= __shfl_sync(0xffffffffu, limit[r / 2], r & 1)) continue;
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[r][i] = fmaf(weight, v[i], acc[r][i]);
      }
    }
  }
};

template <typename T, int kCols, int kRows>
__global__ void __launch_bounds__(SimtShape<kCols>::kWarps * 32, 1) decode_simt_kernel(const __grid_constant__ DecodeParams p, bool vec) {
  using S = SimtShape<kCols>;
  constexpr int kThreads = S::kWarps * 32;
  extern __shared__ __align__(128) float ring[];
  __shared__ long long place[40];
  __shared__ float left_of[S::kWarps][kRows];
  enter_kernel<true>();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Place at = find_place<kThreads>(p, blockIdx.x, 0, place);
  const long long begin = blockIdx.x * at.chunk, end = min(begin + at.chunk, at.units);
  float *stages = ring + warp * kStages * S::kStage;
  for (long long unit = begin; unit < end;) {
    const int keys = seq_keys(p, at.seq);
    const long long seq_units = (long long)p.kv_heads * p.row_blocks * units_of(keys);
    if (unit >= at.first + seq_units) {
      at.first += seq_units;
      ++at.seq;
      continue;
    }
    Piece w;
    unit += next_piece(p, at, blockIdx.x, unit, begin, end, keys, w);

    SimtWarp<T, kCols, kRows> sum;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const T *row = reinterpret_cast<const T *>(p.q.ptr) + row_offset(p, p.q, w, min(r, w.rows - 1));
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int c = col_of<kCols>(lane, i);
        sum.q[r][i] = c < p.head_dim ? to_f32<T>(row[c]) : 0.0f;
        sum.acc[r][i] = 0.0f;
      }
    }
#pragma unroll
    for (int pr = 0; pr < sum.kPairs; ++pr) {
      sum.left[pr] = 0.0;
      sum.limit[pr] = row_limit(p, w.keys, w.row0 + min(2 * pr + (lane & 1), w.rows - 1));
    }
    // the warps' ranges, warp 0 the newest
    const int tiles = (w.k1 - w.k0 + kTileKeys - 1) / kTileKeys, share = (tiles + S::kWarps - 1) / S::kWarps;
    const int t1 = max(tiles - warp * share, 0), t0 = max(t1 - share, 0);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (t1 - 1 - i >= t0)
        bad |= load_stage<T, kCols>(p, w, w.k0 + (t1 - 1 - i) * kTileKeys, w.k1, stages + i * S::kStage, vec);
      cp_async_commit();
    }
    int at_stage = 0;
    for (int t = t1 - 1; t >= t0; --t) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      const int ahead = t - (kStages - 1), into = at_stage == 0 ? kStages - 1 : at_stage - 1;
      if (ahead >= t0) bad |= load_stage<T, kCols>(p, w, w.k0 + ahead * kTileKeys, w.k1, stages + into * S::kStage, vec);
      cp_async_commit();
      sum.tile(p, w, stages + at_stage * S::kStage, w.k0 + t * kTileKeys);
      at_stage = at_stage == kStages - 1 ? 0 : at_stage + 1;
      if (!p.dense) {
        bool gone = true;
#pragma unroll
        for (int pr = 0; pr < sum.kPairs; ++pr) gone = gone && sum.left[pr] < (double)kStickGone * kLn2D;
        if (__all_sync(0xffffffffu, gone)) break;
      }
    }
    cp_async_wait<0>();
    __syncthreads();
    // the warps' sums: each into its own stages' memory, [rows][width], then joined
    if (bad || w.bad) {
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum.acc[r][i] = __int_as_float(0x7fffffff);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < kCols; ++i) stages[r * S::kWidth + col_of<kCols>(lane, i)] = sum.acc[r][i];
#pragma unroll
    for (int pr = 0; pr < sum.kPairs; ++pr)
      if (lane < 2 && 2 * pr + lane < kRows)
        left_of[warp][2 * pr + lane] = bad || w.bad ? __int_as_float(0x7fffffff) : (float)(sum.left[pr] * kLog2eD);
    __syncthreads();
    finish_piece<T, kThreads, S::kWarps, kRows>(p, w, ring, kStages * S::kStage, S::kWidth, 1.0f, left_of);
    __syncthreads();
  }
}

// Joins the pieces of an item that was cut: block c takes the item that begins among the units of the main kernel's block c
// and goes on behind them.
constexpr int kJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ long long place[40];
  enter_kernel<true>();
  if ((int)blockIdx.x >= p.chunks) return;
  const Place at = find_place<kJoinThreads>(p, blockIdx.x + 1, -1, place);
  const long long next = (blockIdx.x + 1) * at.chunk;      // the first unit behind this block's
  if (next >= at.units) return;
  const int n = units_of(seq_keys(p, at.seq));
  const long long in_seq = next - 1 - at.first, first = at.first + in_seq / n * n, last = first + n - 1;
  if (first < next - at.chunk || last < next) return;      // begins earlier; ends here
  Piece w;
  next_piece(p, at, blockIdx.x, first, next - at.chunk, next, seq_keys(p, at.seq), w);
  const int c1 = (int)(last / at.chunk), c0 = blockIdx.x;
  const int parts = p.rows_per_block * p.head_dim;
  for (int e = threadIdx.x; e < w.rows * p.head_dim; e += kJoinThreads) {
    const int r = e / p.head_dim, c = e - r * p.head_dim;
    float o = 0.0f, left = 0.0f;
    for (int i = c1; i >= c0; --i) {
      const long long slot = i == c0 ? 2 * i + 1 : 2 * i;
      const float stick = exp2f(left);
      if (stick == 0.0f) break;
      o += stick * p.part_o[slot * parts + e];
      left += p.part_l[slot * p.rows_per_block + r];
    }
    reinterpret_cast<T *>(p.o.ptr)[row_offset(p, p.o, w, r) + c] = from_f32<T>(o);
  }
  if (threadIdx.x < w.rows) {
    float left = 0.0f;
    for (int i = c1; i >= c0; --i) left += p.part_l[(i == c0 ? 2 * i + 1 : 2 * i) * (long long)p.rows_per_block + threadIdx.x];
    reinterpret_cast<T *>(p.rem)[rem_index(p, w, threadIdx.x)] = from_f32<T>(exp2f(left));
  }
}

template <typename T, int kCols, int kRows> cudaError_t launch_one(const DecodeParams &p, bool vec, cudaStream_t s) {
  using S = SimtShape<kCols>;
  const auto kernel = decode_simt_kernel<T, kCols, kRows>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3(p.chunks), S::kWarps * 32, S::kBytes, s, p, vec);
}
template <typename T, int kCols> cudaError_t launch_rows(const DecodeParams &p, bool vec, cudaStream_t s) {
  switch (p.rows_per_block) {
    case 1: return launch_one<T, kCols, 1>(p, vec, s);
    case 2: return launch_one<T, kCols, 2>(p, vec, s);
    case 4: return launch_one<T, kCols, 4>(p, vec, s);
  }
  if constexpr (kCols <= 4) return launch_one<T, kCols, 8>(p, vec, s);
  return cudaErrorInvalidValue;
}
template <typename T> cudaError_t launch_cols(const DecodeParams &p, cudaStream_t s) {
  auto aligned = [](const PagedRef &t) {
    return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && t.sp % 4 == 0 && t.sh % 4 == 0 && t.st % 4 == 0;
  };
  const bool vec = sizeof(T) == 4 && p.head_dim % 4 == 0 && aligned(p.k) && aligned(p.v);
  if (p.head_dim <= 64) return launch_rows<T, 2>(p, vec, s);
  if (p.head_dim <= 128) return launch_rows<T, 4>(p, vec, s);
  return launch_rows<T, 8>(p, vec, s);
}

}  // namespace

// (More rows of a head_dim over 128 than four do not fit into a thread's registers.)
int decode_simt_rows(int rows, int head_dim) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 || head_dim > 128 ? 4 : 8; }

cudaError_t launch_decode_simt(const DecodeParams &p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case SB_DTYPE_F32: return launch_cols<float>(p, s);
    case SB_DTYPE_BF16: return launch_cols<__nv_bfloat16>(p, s);
    default: return launch_cols<__half>(p, s);
  }
}

cudaError_t launch_decode_join(const DecodeParams &p, int dtype, cudaStream_t s) {
  auto go = [&](auto kernel) { return launch_kernel(kernel, dim3(p.chunks), kJoinThreads, 0, s, p); };
  switch (dtype) {
    case SB_DTYPE_F32: return go(decode_join_kernel<float>);
    case SB_DTYPE_BF16: return go(decode_join_kernel<__nv_bfloat16>);
    default: return go(decode_join_kernel<__half>);
  }
}

}  // namespace sb
