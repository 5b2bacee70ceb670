// Attention of new tokens over a paged key-value cache, tensor-core kernel: bf16 and fp16, rows of whole 16-byte chunks.
//
// What bounds it: every key and value is read once from HBM and takes part in 4 * rows operations per element, `rows` (query
// heads per key head times new tokens) being 1 to 16 here: 1 to 16 operations per byte, where the GPU's ratio is 250.  So the
// kernel is built around the copies: each warp has a ring of 16-key stages of its own, filled with cp.async, and no barrier
// with other warps inside a piece; 192 KiB of stages per SM keep more bytes in flight than the latency of HBM needs (some 50 KiB).
//
// The products are mma.sync ones with the keys as the rows of the tile: S^T = K Q^T, O^T = V^T P^T, 16 keys by 8 queries.  A
// tcgen05 tile takes 64 or 128 rows of one operand from shared memory that whole warps have to hand over; with 8 queries it
// would be no less empty, and the products are not what takes the time.
//
// Row m of the score tile is key 2 m for m < 8, key 2 (m - 8) + 1 otherwise: a thread then holds two neighbouring keys of
// two queries, and the sums over later keys take four shuffles per query.  Base 2 throughout:
//   x = s log2(e) <q, k>,  u = 2^-|x|,  l = log2(1 + u);  log2 beta = min(x, 0) - l,  log2(1 - beta) = -max(x, 0) - l.
// l comes from the series 2 atanh(u / (2 + u)) = 2 (w + w^3 / 3 + w^5 / 5 + ...), to 2^-22 of itself also where u is small: what
// thousands of keys break off adds up.
//
// P enters the second product as the sum of two 16-bit numbers (16 or 22 bits): rounded once it would double the error that the
// output's own rounding makes, and the second product of the pair is free.  In fp16 it is scaled by 2^15, since a weight of 1e-5
// has few bits left there.  Scores, sums and the output's accumulators are 32-bit, the stick between tiles 64-bit.
#include "sb_decode.cuh"
#include "sb_ptx.cuh"

namespace sb {

namespace {

using ptx::ex2;
using ptx::rcp;
using ptx::smem_u32;

// kD: head_dim rounded up to 64, 128, 256; kN: blocks of 8 query rows.  As many warps as their registers allow: a tile is a
// chain of some 800 cycles (scores, scan over keys, weights, values), and other warps' tiles are what fills them.
template <int kD, int kN> struct TcShape {
  static constexpr int kChunks = kD / 8;                            // 16-byte chunks of a row
  static constexpr int kHalf = kTileKeys * kD * 2;                  // bytes of a stage's keys (or values)
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kWarps = kD == 256 ? 6 : kD / 64 * kN <= 2 ? 12 : 8;
  static constexpr int kStages = 192 * 1024 / (kWarps * kStage);
  static constexpr int kBytes = kWarps * kStages * kStage;          // 192 KiB
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t x);
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
template <typename T> constexpr float kScaleP = 1.0f;
template <> constexpr float kScaleP<__half> = 32768.0f;

// (ptx::ex2 gives 0 for what is below 2^-126; weights go down to 2^-149, where the stick counts as used up)
__device__ __forceinline__ float weight(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2(1 + u), 0 <= u <= 1; NaN for NaN.
__device__ __forceinline__ float log2_1p(float u) {
  const float w = u * rcp(2.0f + u), t = w * w;
  float s = fmaf(t, 1.0f / 11, 1.0f / 9);
  s = fmaf(t, s, 1.0f / 7);
  s = fmaf(t, s, 1.0f / 5);
  s = fmaf(t, s, 1.0f / 3);
  s = fmaf(t, s, 1.0f);
  return 2.0f * kLog2e * w * s;
}

// Where chunk c of row r of a stage's keys or values lies: the eight even (or odd) rows that one ldmatrix reads are in eight
// different places of the 128 bytes that the banks span.
template <int kD> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)(r * kD * 2 + ((c ^ ((r >> 1) & 7)) << 4));
}

// The tensor-core engine.  kN: blocks of 8 query rows.
template <typename T, int kD, int kN> struct TcEngine : TcShape<kD, kN> {
  using S = TcShape<kD, kN>;
  using S::kHalf;
  uint32_t q[kN][kD / 16][2];
  float acc[kD / 16][kN][4];
  double left[kN][2];
  int limit[kN][2];
  bool real[kN][2];

  __device__ static __forceinline__ void prefetch_rows(const DecodeParams &p, const Piece &w) { prefetch_q(p, w, 2); }

  // 16 rows from slot `slot` of one page on; columns behind head_dim are zeros.
  __device__ static __forceinline__ void copy_run(const DecodeParams &p, const Piece &w, int page, int slot, char *to) {
    const int lane = threadIdx.x & 31;
    constexpr int kAtOnce = 32 / S::kChunks;     // rows of one instruction
    const int c = lane % S::kChunks, r0 = lane / S::kChunks;
    const bool col = c * 8 < p.head_dim;
    const char *k = p.k.ptr + (page * p.k.sp + w.head * p.k.sh + (slot + r0) * p.k.st) * 2 + (col ? c * 16 : 0);
    const char *v = p.v.ptr + (page * p.v.sp + w.head * p.v.sh + (slot + r0) * p.v.st) * 2 + (col ? c * 16 : 0);
    const long long k_step = kAtOnce * 2 * p.k.st, v_step = kAtOnce * 2 * p.v.st;
    const uint32_t stage = smem_u32(to);
#pragma unroll
    for (int i = 0; i < kTileKeys / kAtOnce; ++i) {
      const uint32_t at = stage + chunk_at<kD>(i * kAtOnce + r0, c);
      cp_async16(at, k + i * k_step, col);
      cp_async16(at + kHalf, v + i * v_step, col);
    }
  }
  // Lane l has the page (-1: none, zeros) and slot of row l & 15.
  __device__ static __forceinline__ void copy(const DecodeParams &p, const Piece &w, int page, int slot, char *to) {
    const int lane = threadIdx.x & 31;
    const bool value = lane >= 16;               // lanes 16..31 hold the values' offsets
    const PagedRef &t = value ? p.v : p.k;
    const long long at = page < 0 ? -1 : (page * t.sp + w.head * t.sh + slot * t.st) * 2;
    constexpr int kAtOnce = 32 / S::kChunks;
    const int c = lane % S::kChunks, r0 = lane / S::kChunks;
    const bool col = c * 8 < p.head_dim;
    const uint32_t stage = smem_u32(to);
#pragma unroll
    for (int i = 0; i < kTileKeys / kAtOnce; ++i) {
      const int r = i * kAtOnce + r0;
      const long long ak = __shfl_sync(0xffffffffu, at, r), av = __shfl_sync(0xffffffffu, at, r + 16);
      const bool take = ak >= 0 && col;
      cp_async16(stage + chunk_at<kD>(r, c), take ? p.k.ptr + ak + c * 16 : p.k.ptr, take);
      cp_async16(stage + kHalf + chunk_at<kD>(r, c), take ? p.v.ptr + av + c * 16 : p.v.ptr, take);
    }
  }

  __device__ __forceinline__ void start(const DecodeParams &p, const Piece &w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = n * 8 + g;
      const char *row = p.q.ptr + 2 * row_offset(p, p.q, w.seq, w.head, w.row0 + min(r, w.rows - 1));
#pragma unroll
      for (int i = 0; i < kD / 16; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c = i * 16 + half * 8 + t * 2;
          q[n][i][half] = r < w.rows && c < p.head_dim ? *reinterpret_cast<const uint32_t *>(row + 2 * c) : 0;
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int query = n * 8 + t * 2 + j;
        left[n][j] = 0.0;
        real[n][j] = query < w.rows;
        limit[n][j] = row_limit(p, w.keys, w.row0 + min(query, w.rows - 1));
      }
#pragma unroll
      for (int i = 0; i < kD / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
    }
  }

  // O^T += V^T P^T, P as two 16-bit numbers; `b`: [row block][keys 2 m, 2 m + 1][high, low].  kSome: only for the queries whose
  // limits are in [low, high).
  template <bool kSome> __device__ __forceinline__ void add_values(uint32_t values, const uint32_t (&b)[kN][2][2], int low, int high) {
    const int lane = threadIdx.x & 31;
    const int r = 2 * (lane & 7) + (lane >> 4), c = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < kD / 16; ++i) {
      uint32_t a[4];
      ldsm4_t(values + chunk_at<kD>(r, 2 * i + c), a);
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = acc[i][n][j];
        mma<T>(o, a, b[n][0][0], b[n][1][0]);
        mma<T>(o, a, b[n][0][1], b[n][1][1]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!kSome || (limit[n][j & 1] >= low && limit[n][j & 1] < high)) acc[i][n][j] = o[j];
      }
    }
  }

  __device__ __forceinline__ void tile(const DecodeParams &p, const Piece &w, char *to, int key0) {
    const uint32_t stage = smem_u32(to);
    const int lane = threadIdx.x & 31, g = lane >> 2;
    float s[kN][4], odd[kN][4];           // two chains of products
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = odd[n][j] = 0.0f;
    {
      const int r = 2 * (lane & 7) + ((lane >> 3) & 1), c = lane >> 4;
#pragma unroll
      for (int i = 0; i < kD / 16; ++i) {
        uint32_t a[4];
        ldsm4(stage + chunk_at<kD>(r, 2 * i + c), a);
#pragma unroll
        for (int n = 0; n < kN; ++n) mma<T>(i & 1 ? odd[n] : s[n], a, q[n][i][0], q[n][i][1]);
      }
    }
    const float scale = p.scale * kLog2e;
    float a[kN][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {                  // queries 2 t + j; keys 2 g (s[n][j]) and 2 g + 1 (s[n][2 + j])
        float beta[2], broken[2];
#pragma unroll
        for (int key = 0; key < 2; ++key) {
          const float x = (s[n][2 * key + j] + odd[n][2 * key + j]) * scale, l = log2_1p(ex2(-fabsf(x)));
          const bool in = key0 + 2 * g + key < limit[n][j];
          beta[key] = in ? fminf(x, 0.0f) - l : -INFINITY;
          broken[key] = in ? -(fmaxf(x, 0.0f) + l) : 0.0f;
          if (in && x != x) beta[key] = broken[key] = x;      // (fminf and fmaxf drop a NaN)
        }
        const float both = broken[0] + broken[1];
        float later = __shfl_down_sync(0xffffffffu, both, 4);
        if (g == 7) later = 0.0f;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          const float other = __shfl_down_sync(0xffffffffu, later, d);
          if (lane + d < 32) later += other;
        }
        const float base = (float)left[n][j] + later;
        a[n][2 + j] = weight(beta[1] + base) * kScaleP<T>;
        a[n][j] = weight(beta[0] + (base + broken[1])) * kScaleP<T>;
        left[n][j] += (double)__shfl_sync(0xffffffffu, later + both, lane & 3);
      }
    }
    // the two 16-bit parts of the weights, moved from (key, query) to (query, key)
    uint32_t b[kN][2][2];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int key = 0; key < 2; ++key) {
        const uint32_t hi = pack<T>(a[n][2 * key], a[n][2 * key + 1]);
        const float2 back = unpack<T>(hi);
        b[n][key][0] = transpose8x8(hi);
        b[n][key][1] = transpose8x8(pack<T>(a[n][2 * key] - back.x, a[n][2 * key + 1] - back.y));
      }
    const uint32_t values = stage + kHalf;
    if (key0 + kTileKeys <= w.edge) {
      add_values<false>(values, b, 0, 0);
      return;
    }
    // Some rows do not attend to some keys of the tile.  Those keys' values are taken out, not multiplied by 0 (they may be no
    // numbers): the rows take their turns from the longest reach down, and the values that are out of reach become zeros.
    add_values<true>(values, b, key0 + kTileKeys, 0x7fffffff);
    for (int reach = min(w.k1, key0 + kTileKeys - 1); reach >= max(w.edge, key0 + 1); --reach) {
      __syncwarp();
      if (lane < S::kChunks)
        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(values + chunk_at<kD>(reach - key0, lane)), "r"(0) : "memory");
      __syncwarp();
      add_values<true>(values, b, reach, reach + 1);
    }
  }

  __device__ __forceinline__ bool gone() const {
    bool all = true;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) all = all && (!real[n][j] || left[n][j] < (double)kStickGone);
    return __all_sync(0xffffffffu, all);
  }

  __device__ __forceinline__ void finish(const DecodeParams &p, const Piece &w, int slot, bool bad) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float nan = __int_as_float(0x7fffffff);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = n * 8 + t * 2 + j;
        if (r >= w.rows) continue;
        const RowOut<T> out(p, w, slot, r);
#pragma unroll
        for (int i = 0; i < kD / 16; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c = i * 16 + half * 8 + g;
            if (c < p.head_dim) out.put(c, bad ? nan : acc[i][n][half * 2 + j] * (1.0f / kScaleP<T>));
          }
        if (g == 0) put_rem<T>(p, w, slot, r, bad ? nan : (float)left[n][j]);
      }
  }
};

template <typename T, int kD, int kN>
__global__ void __launch_bounds__(TcShape<kD, kN>::kWarps * 32, 1) decode_tc_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) char ring[];
  __shared__ ChunkShared<TcShape<kD, kN>::kWarps> shared;
  enter_kernel<true>();
  decode_chunks<TcEngine<T, kD, kN>>(p, ring, shared);
}

template <typename T, int kD, int kN> cudaError_t launch_one(const DecodeParams &p, cudaStream_t s) {
  using S = TcShape<kD, kN>;
  const auto kernel = decode_tc_kernel<T, kD, kN>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3(p.chunks / S::kWarps), S::kWarps * 32, S::kBytes, s, p);
}
template <typename T> cudaError_t launch_shape(const DecodeParams &p, cudaStream_t s) {
  const int n = p.rows_per_block / 8;
  if (p.head_dim <= 64) return n == 1 ? launch_one<T, 64, 1>(p, s) : n == 2 ? launch_one<T, 64, 2>(p, s) : launch_one<T, 64, 4>(p, s);
  if (p.head_dim <= 128) return n == 1 ? launch_one<T, 128, 1>(p, s) : launch_one<T, 128, 2>(p, s);
  return launch_one<T, 256, 1>(p, s);
}

}  // namespace

// Query rows per item, as many as a thread's 64 accumulators hold; the keys are read once for them.
int decode_tc_rows(int rows, int head_dim) {
  const int most = head_dim <= 64 ? 32 : head_dim <= 128 ? 16 : 8;
  return rows <= 8 || most == 8 ? 8 : rows <= 16 || most == 16 ? 16 : 32;
}
int decode_tc_warps(int rows, int head_dim) {
  if (head_dim > 128) return TcShape<256, 1>::kWarps;
  if (head_dim > 64) return rows == 8 ? TcShape<128, 1>::kWarps : TcShape<128, 2>::kWarps;
  return rows == 8 ? TcShape<64, 1>::kWarps : rows == 16 ? TcShape<64, 2>::kWarps : TcShape<64, 4>::kWarps;
}

cudaError_t launch_decode_tc(const DecodeParams &p, int dtype, cudaStream_t s) {
  return dtype == SB_DTYPE_BF16 ? launch_shape<__nv_bfloat16>(p, s) : launch_shape<__half>(p, s);
}

}  // namespace sb
