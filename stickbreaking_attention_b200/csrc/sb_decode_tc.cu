// Attention of new tokens over a paged key-value cache, tensor-core kernel: bf16 and fp16, rows of whole 16-byte chunks.
//
// What bounds it: every key and value is read once from HBM and takes part in 4 * rows operations per element.  With `rows` (query
// heads per key head times new tokens) of 1 to 16 that is 1 to 16 operations per byte, where the GPU's ratio is 250.  (More rows
// are taken 16, or 8 or 32, at a time, for each of which all keys are read again, through L2: 16 / 4 heads, 8192 tokens and 64, 256, 1024
// new ones take 68, 200, 724 us, 63 to 95 TFLOP/s.)  So the kernel is built around the copies: each warp has a ring of 16-key stages of its own, filled with cp.async, and no barrier with
// other warps; 192 KiB of stages per SM keep more bytes in flight than the latency of HBM needs (some 50 KiB).  (TMA, boxes of 64
// columns x 16 rows issued by one lane, took the same time to within 2 %, its longer latency weighing as much as the instructions that it saves.)
//
// The products are mma.sync ones with the keys as the rows of the tile: S^T = K Q^T, O^T = V^T P^T, 16 keys by 8 queries.  A
// tcgen05 tile takes 64 or 128 rows of one operand from shared memory that whole warps have to hand over; with 8 queries it
// would be no less empty, and the products are not what takes the time.
//
// A thread holds rows g and g + 8 of the score tile.  They are keys 2 g and 2 g + 1 of the 16 (for g >= 4 the other way round), so
// that the products over later keys take four shuffles per query; and the eight rows that one ldmatrix reads are eight different
// ones modulo 8, which is what the swizzle needs to put them into different banks.  No logarithms:
//   x = s log2(e) <q, k>,  e = 2^-|x|,  1 - beta = 1 / (1 + 2^x) = (e or 1) / (1 + e),  beta = (1 or e) / (1 + e)  (x >= 0 or not),
//   weight = stick * (product of 1 - beta over the tile's later keys) * beta,
// and the stick behind the tile is what was there less the tile's weights, where more than 7/8 of it are left, else the product.  The
// difference loses nothing over thousands of keys that take 1e-5 each, whose 1 - beta are rounded in their last bits; the
// product loses nothing where little is left.  The tile's weights are added up by one more product, with ones for values, as
// 16-bit numbers, whose steps have an end: a stick below 2^-16 in fp16, 2^-100 in bf16, is the product always, or it would stand still
// where a tile's weights are 0 in 16 bits.  (The last bits of 1 - beta, 2^-21 of the stick per tile, are then as much as the steps of
// 2^-39 of 16 weights, and of a share of 2^-16 of the whole.)  Below 2^-100 it is rounded down, so that it comes to 0
// instead of standing still at fp32's smallest numbers.
//
// P enters the second product as the sum of 16-bit numbers: three in bf16 (24 bits, as many as the weights have) and two in fp16
// (22 bits).  Up to four query rows leave columns of a product empty, and the parts of the weights take these: one product for
// one or two rows, two (bf16) or one (fp16) for up to four.  In bf16 two parts, 16 bits, in two products took 154.3 us for 154.9
// (64 sequences x 16 heads x 512..4096 tokens), 89.6 for 91.3 (48 ragged ones, 4 query heads to a key head), 62.9 for 58.8 (32 of 256 columns);
// the share of output values that are not the nearest of their type to the exact one was 2.6e-3 for 6.5e-4 (32-bit CUDA cores: 5.7e-4) in
// the first, 1.9e-3 for 4.2e-4 in the second.  In fp16 weights are scaled by 2^15 and so held in steps of 2^-39: each is off by up to 2^-40.
// Scores, weights and the output's accumulators are 32-bit, the stick 32-bit with what its sums lost.
#include "sb_decode.cuh"
#include "sb_ptx.cuh"

namespace sb {

namespace {

using ptx::ex2;
using ptx::rcp;
using ptx::smem_u32;

// kD: head_dim rounded up to 64, 128, 256; kN: blocks of 8 query rows.  As many warps as their registers allow: a tile is a
// chain of some 700 cycles (scores, scan over keys, weights, values), and other warps' tiles are what fills them.  Times in us with
// 8, 10, 12, 16 warps.  128 columns, 8 rows: 64 sequences x 16 heads x 512..4096 tokens 153, 153, 155, 148; 48 ragged sequences of
// shared key heads, half of them local, 119, 114, 91, 94; one of 131072 tokens 56, 57, 57, 59.  64 columns, 8 rows: 64 x 16 x 512..4096 117, 105, 83, 84;
// 16 rows: 24 sequences with 4 new tokens 29.5, 29.9, 28.5, 32.6.  With 12 warps a thread has 168 registers, which 64 columns and 16 rows
// overrun by 4 (fp16) or 7 (bf16), with 16 it has 128, which these and 128 columns overrun by 4 to 26.
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
template <typename T> constexpr uint32_t kOnes = 0x3f803f80;      // two times 1.0
template <> constexpr uint32_t kOnes<__half> = 0x3c003c00;
template <typename T> constexpr float kSmallStick = 0x1p-100f;     // from here on the difference is not taken
template <> constexpr float kSmallStick<__half> = 0x1p-16f;
template <typename T> constexpr int kParts = 3;                    // 16-bit numbers that make up a weight
template <> constexpr int kParts<__half> = 2;

// Where chunk c of row r of a stage's keys or values lies: blocks of 64 columns, rows of 128 bytes, swizzled.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * (kTileKeys * 128) + r * 128 + (((c ^ r) & 7) << 4));
}
// The key of the tile that row g (second false) or g + 8 of a product's operand is.
__device__ __forceinline__ int key_of(int g, bool second) { return 2 * g + (second != (g >= 4)); }

// The tensor-core engine.  kN: blocks of 8 query rows.  kSets: where the rows are few (kN 1) they are in the 8 columns of the products
// kSets times, and each set of columns has a part of the weights of its own in one product; the sets' sums are added up at the end.
template <typename T, int kD, int kN, int kSets> struct TcEngine : TcShape<kD, kN> {
  using S = TcShape<kD, kN>;
  using S::kHalf;
  static_assert(kSets == 1 || kN == 1, "");
  static constexpr int kOfSet = kN * 8 / kSets;                              // rows of a set; a thread's two columns are in the same one
  static constexpr int kPasses = (kParts<T> + kSets - 1) / kSets;            // products that the parts of the weights take
  uint32_t q[kN][kD / 16][2];
  float acc[kD / 16][kN][4];
  LongSum stick[kN][2];
  int limit[kN][2];
  bool real[kN][2];

  __device__ static __forceinline__ void prefetch_rows(const DecodeParams &p, const Piece &w) { prefetch_q(p, w, 2); }

  // What the sets of columns sum up to, in all of them.  (In the same order in each: the sets of a row stay the same.)
  __device__ static __forceinline__ float over_sets(float x) {
#pragma unroll
    for (int d = kOfSet / 2; d < 4; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
  }

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
      const uint32_t at = stage + chunk_at(i * kAtOnce + r0, c);
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
      cp_async16(stage + chunk_at(r, c), take ? p.k.ptr + ak + c * 16 : p.k.ptr, take);
      cp_async16(stage + kHalf + chunk_at(r, c), take ? p.v.ptr + av + c * 16 : p.v.ptr, take);
    }
  }

  __device__ __forceinline__ void start(const DecodeParams &p, const Piece &w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = (n * 8 + g) % kOfSet;
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
        const int query = (n * 8 + t * 2 + j) % kOfSet;
        stick[n][j] = LongSum{1.0f, 0.0f};
        real[n][j] = query < w.rows;
        limit[n][j] = row_limit(p, w.keys, w.row0 + min(query, w.rows - 1));
      }
#pragma unroll
      for (int i = 0; i < kD / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
    }
  }

  // O^T += V^T P^T; `b`: the weights, [row block][rows m, m + 8][product].  kSome: only for the queries whose limits are in
  // [low, high).
  template <bool kSome> __device__ __forceinline__ void add_values(uint32_t values, const uint32_t (&b)[kN][2][kPasses], int low, int high) {
    const int lane = threadIdx.x & 31;
    const int r = key_of(lane & 7, lane >> 4), c = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < kD / 16; ++i) {
      uint32_t a[4];
      ldsm4_t(values + chunk_at(r, 2 * i + c), a);
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = acc[i][n][j];
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) mma<T>(o, a, b[n][0][pass], b[n][1][pass]);
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
      const int r = key_of(lane & 7, lane >> 3 & 1), c = lane >> 4;
#pragma unroll
      for (int i = 0; i < kD / 16; ++i) {
        uint32_t a[4];
        ldsm4(stage + chunk_at(r, 2 * i + c), a);
#pragma unroll
        for (int n = 0; n < kN; ++n) mma<T>(i & 1 ? odd[n] : s[n], a, q[n][i][0], q[n][i][1]);
      }
    }
    const float scale = p.scale * kLog2e;
    const bool edge = key0 + kTileKeys > w.edge;     // some rows do not attend to some keys
    float a[kN][4], rest[kN][2];                     // weights; product of 1 - beta over the tile
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {                  // queries 2 t + j; rows g (s[n][j]) and g + 8 (s[n][2 + j])
        float beta[2], kept[2];
#pragma unroll
        for (int row = 0; row < 2; ++row) {
          const float x = (s[n][2 * row + j] + odd[n][2 * row + j]) * scale, e = ex2(-fabsf(x)), d = rcp(1.0f + e), ed = e * d;
          beta[row] = x >= 0.0f ? d : ed;            // (NaN: both are)
          kept[row] = x >= 0.0f ? ed : d;
        }
        if (edge) {
#pragma unroll
          for (int row = 0; row < 2; ++row)
            if (key0 + key_of(g, row) >= limit[n][j]) {
              beta[row] = 0.0f;
              kept[row] = 1.0f;
            }
        }
        const float both = kept[0] * kept[1];
        float later = __shfl_down_sync(0xffffffffu, both, 4);
        if (g == 7) later = 1.0f;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          const float other = __shfl_down_sync(0xffffffffu, later, d);
          if (lane + d < 32) later *= other;
        }
        rest[n][j] = __shfl_sync(0xffffffffu, later * both, lane & 3);
        const float whole = stick[n][j].sum * kScaleP<T> * later;
        a[n][j] = beta[0] * (g < 4 ? whole * kept[1] : whole);          // the older key of the two comes behind the newer one
        a[n][2 + j] = beta[1] * (g < 4 ? whole : whole * kept[0]);
      }
    }
    // the 16-bit parts of the weights, the largest first, part i in set i % kSets of product i / kSets, moved from (key, query) to
    // (query, key)
    uint32_t b[kN][2][kPasses];
    const int set = (lane & 3) * 2 / kOfSet;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int row = 0; row < 2; ++row) {
        uint32_t own[kPasses] = {};
#pragma unroll
        for (int part = 0; part < kParts<T>; ++part) {
          const uint32_t rounded = pack<T>(a[n][2 * row], a[n][2 * row + 1]);
          const float2 back = unpack<T>(rounded);
          a[n][2 * row] -= back.x;               // what is left for the parts behind this one, exactly
          a[n][2 * row + 1] -= back.y;
          if (kSets == 1 || set == part % kSets) own[part / kSets] = rounded;
        }
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) b[n][row][pass] = transpose8x8(own[pass]);
      }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const uint32_t ones[4] = {kOnes<T>, kOnes<T>, kOnes<T>, kOnes<T>};
      float sum[4] = {};                             // [j]: all weights of query 2 t + j
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) mma<T>(sum, ones, b[n][0][pass], b[n][1][pass]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float whole = stick[n][j].sum, taken = over_sets(sum[j]);
        if (rest[n][j] > 0.875f && whole > kSmallStick<T>) stick[n][j].add(taken * (-1.0f / kScaleP<T>));
        else stick[n][j] = LongSum{whole > 0x1p-100f ? whole * rest[n][j] : __fmul_rz(whole, rest[n][j]), 0.0f};
      }
    }
    const uint32_t values = stage + kHalf;
    if (!edge) {
      add_values<false>(values, b, 0, 0);
      return;
    }
    // Some rows do not attend to some keys of the tile.  Those keys' values are taken out, not multiplied by 0 (they may be no
    // numbers): the rows take their turns from the longest reach down, and the values that are out of reach become zeros.
    const auto clear = [&](int row) {
      if (lane < S::kChunks)
        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(values + chunk_at(row, lane)), "r"(0) : "memory");
    };
    if (w.k1 >= key0 + kTileKeys) add_values<true>(values, b, key0 + kTileKeys, 0x7fffffff);
    for (int key = w.k1 + 1; key < key0 + kTileKeys; ++key) clear(key - key0);
    for (int reach = min(w.k1, key0 + kTileKeys - 1); reach >= max(w.edge, key0 + 1); --reach) {
      __syncwarp();
      clear(reach - key0);
      __syncwarp();
      add_values<true>(values, b, reach, reach + 1);
    }
  }

  __device__ __forceinline__ bool gone() const {
    bool all = true;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) all = all && (!real[n][j] || stick[n][j].sum == 0.0f);
    return __all_sync(0xffffffffu, all);
  }

  // A piece that is not the whole item leaves its accumulators as they lie in the registers, 16 bytes a lane, for the join kernel.
  __device__ __forceinline__ void finish(const DecodeParams &p, const Piece &w, int slot, bool bad) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float nan = __int_as_float(0x7fffffff);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kD / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] = over_sets(acc[i][n][j]);
    if (bad) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < kD / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][n][j] = nan;
        stick[n][0].sum = stick[n][1].sum = nan;
      }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = n * 8 + t * 2;
      if (r >= w.rows) continue;
      if (slot < 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (r + j >= w.rows) continue;
          T *const out = reinterpret_cast<T *>(p.o.ptr) + row_offset(p, p.o, w.seq, w.head, w.row0 + r + j);
#pragma unroll
          for (int i = 0; i < kD / 16; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int c = i * 16 + half * 8 + g;
              if (c < p.head_dim) out[c] = from_f32<T>(acc[i][n][half * 2 + j] * (1.0f / kScaleP<T>));
            }
          if (g == 0) reinterpret_cast<T *>(p.rem)[rem_index(p, w.seq, w.head, w.row0 + r + j)] = from_f32<T>(stick[n][j].sum);
        }
      } else {
        float4 *const part = reinterpret_cast<float4 *>(p.part_o + (long long)slot * (kN * 8 * kD)) + n * (kD / 16) * 32 + lane;
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) part[i * 32] = make_float4(acc[i][n][0], acc[i][n][1], acc[i][n][2], acc[i][n][3]);
        if (g == 0) *reinterpret_cast<float2 *>(p.part_l + (long long)slot * (kN * 8) + r) = make_float2(stick[n][0].sum, stick[n][1].sum);
      }
    }
  }
};

template <typename T, int kD, int kN, int kSets>
__global__ void __launch_bounds__(TcShape<kD, kN>::kWarps * 32, 1) decode_tc_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) char ring[];
  __shared__ ChunkShared<TcShape<kD, kN>::kWarps> shared;
  enter_kernel<true>();
  decode_chunks<TcEngine<T, kD, kN, kSets>>(p, ring, shared);
}

// Joins the pieces of the items that were cut, newest first, 8 rows x 16 columns at a time as a warp's registers held them: a lane has two
// rows and two columns.  Each warp has such a part of its own (kTogether 1), or kTogether warps have the same one and take a run
// of its pieces each, whose sums are joined like pieces.
constexpr int kJoinDeep = 8;
// Eight pieces in flight together.  (One statement: left to itself the compiler loads a few, adds them up, and only then loads the
// next, which is a trip to L2 each.)
__device__ __forceinline__ void load_eight(const float4 *const (&at)[8], float4 (&x)[8]) {
  asm volatile(
      "ld.global.v4.f32 {%0,%1,%2,%3}, [%32];\n\tld.global.v4.f32 {%4,%5,%6,%7}, [%33];\n\t"
      "ld.global.v4.f32 {%8,%9,%10,%11}, [%34];\n\tld.global.v4.f32 {%12,%13,%14,%15}, [%35];\n\t"
      "ld.global.v4.f32 {%16,%17,%18,%19}, [%36];\n\tld.global.v4.f32 {%20,%21,%22,%23}, [%37];\n\t"
      "ld.global.v4.f32 {%24,%25,%26,%27}, [%38];\n\tld.global.v4.f32 {%28,%29,%30,%31}, [%39];"
      : "=f"(x[0].x), "=f"(x[0].y), "=f"(x[0].z), "=f"(x[0].w), "=f"(x[1].x), "=f"(x[1].y), "=f"(x[1].z), "=f"(x[1].w),
        "=f"(x[2].x), "=f"(x[2].y), "=f"(x[2].z), "=f"(x[2].w), "=f"(x[3].x), "=f"(x[3].y), "=f"(x[3].z), "=f"(x[3].w),
        "=f"(x[4].x), "=f"(x[4].y), "=f"(x[4].z), "=f"(x[4].w), "=f"(x[5].x), "=f"(x[5].y), "=f"(x[5].z), "=f"(x[5].w),
        "=f"(x[6].x), "=f"(x[6].y), "=f"(x[6].z), "=f"(x[6].w), "=f"(x[7].x), "=f"(x[7].y), "=f"(x[7].z), "=f"(x[7].w)
      : "l"(at[0]), "l"(at[1]), "l"(at[2]), "l"(at[3]), "l"(at[4]), "l"(at[5]), "l"(at[6]), "l"(at[7])
      : "memory");
}
__device__ __forceinline__ void load_eight(const float2 *const (&at)[8], float2 (&x)[8]) {
  asm volatile(
      "ld.global.v2.f32 {%0,%1}, [%16];\n\tld.global.v2.f32 {%2,%3}, [%17];\n\tld.global.v2.f32 {%4,%5}, [%18];\n\tld.global.v2.f32 {%6,%7}, [%19];\n\t"
      "ld.global.v2.f32 {%8,%9}, [%20];\n\tld.global.v2.f32 {%10,%11}, [%21];\n\tld.global.v2.f32 {%12,%13}, [%22];\n\tld.global.v2.f32 {%14,%15}, [%23];"
      : "=f"(x[0].x), "=f"(x[0].y), "=f"(x[1].x), "=f"(x[1].y), "=f"(x[2].x), "=f"(x[2].y), "=f"(x[3].x), "=f"(x[3].y),
        "=f"(x[4].x), "=f"(x[4].y), "=f"(x[5].x), "=f"(x[5].y), "=f"(x[6].x), "=f"(x[6].y), "=f"(x[7].x), "=f"(x[7].y)
      : "l"(at[0]), "l"(at[1]), "l"(at[2]), "l"(at[3]), "l"(at[4]), "l"(at[5]), "l"(at[6]), "l"(at[7])
      : "memory");
}
// Adds a run of keys (x, l) behind what is summed up in (o, left).  (0 times what is no number stays out.)
__device__ __forceinline__ void add_behind(float4 &o, float2 &left, const float4 &x, const float2 &l) {
  o.x += left.x != 0.0f ? left.x * x.x : 0.0f;
  o.y += left.y != 0.0f ? left.y * x.y : 0.0f;
  o.z += left.x != 0.0f ? left.x * x.z : 0.0f;
  o.w += left.y != 0.0f ? left.y * x.w : 0.0f;
  left.x = left.x != 0.0f ? left.x * l.x : 0.0f;
  left.y = left.y != 0.0f ? left.y * l.y : 0.0f;
}

template <typename T, int kWarps, int kTogether>
__global__ void __launch_bounds__(kWarps * 32) decode_tc_join_kernel(const __grid_constant__ DecodeParams p) {
  enter_kernel<true>();
  const int4 note = p.notes[blockIdx.x];
  if (note.w == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / kTogether, member = warp % kTogether;
  const int head = p.row_blocks == 1 ? note.y : note.y / p.row_blocks, row0 = (note.y - head * p.row_blocks) * p.rows_per_block;
  const int rows = min(p.rows - row0, p.rows_per_block), blocks = p.part_cols / 16;
  const int job = blockIdx.y * (kWarps / kTogether) + team, n = job / blocks, i = job - n * blocks;
  const int r = n * 8 + (lane & 3) * 2, c = i * 16 + (lane >> 2);
  const bool real = r < rows && i * 16 < p.head_dim;      // (columns behind head_dim are there, as zeros)
  const int share = (note.w + kTogether - 1) / kTogether;
  const int begin = min(member * share, note.w), end = min(begin + share, note.w);
  // k-th piece from the newest on: the oldest is its chunk's last, the others are their chunk's first
  const auto slot_of = [&](int k) { return 2LL * (note.z + note.w - 1 - k) + (k == note.w - 1 ? 1 : 0); };
  const int slot_size = p.rows_per_block * p.part_cols;
  const float4 *const parts = reinterpret_cast<const float4 *>(p.part_o) + job * 32 + lane;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float2 left = make_float2(1.0f, 1.0f);       // of the stick
  if (real) {
    for (int k0 = begin; k0 < end; k0 += kJoinDeep) {
      const float4 *at[kJoinDeep];
      const float2 *l_at[kJoinDeep];
      float4 x[kJoinDeep];
      float2 l[kJoinDeep];
#pragma unroll
      for (int k = 0; k < kJoinDeep; ++k) {
        const long long slot = slot_of(min(k0 + k, end - 1));
        at[k] = parts + slot * (slot_size / 4);
        l_at[k] = reinterpret_cast<const float2 *>(p.part_l + slot * p.rows_per_block + r);
      }
      load_eight(at, x);
      load_eight(l_at, l);
#pragma unroll
      for (int k = 0; k < kJoinDeep; ++k)
        if (k0 + k < end) add_behind(o, left, x[k], l[k]);
    }
  }
  if constexpr (kTogether > 1) {
    __shared__ float4 sums[kWarps][32];
    __shared__ float2 lefts[kWarps][32];
    sums[warp][lane] = o;
    lefts[warp][lane] = left;
    __syncthreads();
    if (member != 0) return;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    left = make_float2(1.0f, 1.0f);
#pragma unroll 8
    for (int m = 0; m < kTogether; ++m) add_behind(o, left, sums[warp + m][lane], lefts[warp + m][lane]);
  }
  if (!real) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (r + j >= rows) break;
    T *const out = reinterpret_cast<T *>(p.o.ptr) + row_offset(p, p.o, note.x, head, row0 + r + j);
    if (c < p.head_dim) out[c] = from_f32<T>((j ? o.y : o.x) * (1.0f / kScaleP<T>));
    if (c + 8 < p.head_dim) out[c + 8] = from_f32<T>((j ? o.w : o.z) * (1.0f / kScaleP<T>));
    if (c == 0) reinterpret_cast<T *>(p.rem)[rem_index(p, note.x, head, row0 + r + j)] = from_f32<T>(j ? left.y : left.x);
  }
}

template <typename T, int kD, int kN, int kSets = 1> cudaError_t launch_one(const DecodeParams &p, cudaStream_t s) {
  using S = TcShape<kD, kN>;
  const auto kernel = decode_tc_kernel<T, kD, kN, kSets>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3(p.chunks / S::kWarps), S::kWarps * 32, S::kBytes, s, p);
}
// Eight rows or fewer: as many sets as there is room for and parts of the weights to put there.
template <typename T, int kD> cudaError_t launch_few(const DecodeParams &p, cudaStream_t s) {
  if (kParts<T> > 2 && p.rows <= 2) return launch_one<T, kD, 1, kParts<T> == 2 ? 2 : 4>(p, s);
  return p.rows <= 4 ? launch_one<T, kD, 1, 2>(p, s) : launch_one<T, kD, 1>(p, s);
}
template <typename T> cudaError_t launch_shape(const DecodeParams &p, cudaStream_t s) {
  const int n = p.rows_per_block / 8;
  if (p.head_dim <= 64) return n == 1 ? launch_few<T, 64>(p, s) : n == 2 ? launch_one<T, 64, 2>(p, s) : launch_one<T, 64, 4>(p, s);
  if (p.head_dim <= 128) return n == 1 ? launch_few<T, 128>(p, s) : launch_one<T, 128, 2>(p, s);
  return launch_few<T, 256>(p, s);
}

}  // namespace

// Query rows per item, as many as a thread's 64 accumulators hold; the keys are read once for them.
int decode_tc_rows(int rows, int head_dim) {
  const int most = head_dim <= 64 ? 32 : head_dim <= 128 ? 16 : 8;
  return rows <= 8 || most == 8 ? 8 : rows <= 16 || most == 16 ? 16 : 32;
}
int decode_tc_cols(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
int decode_tc_warps(int rows, int head_dim) {
  if (head_dim > 128) return TcShape<256, 1>::kWarps;
  if (head_dim > 64) return rows == 8 ? TcShape<128, 1>::kWarps : TcShape<128, 2>::kWarps;
  return rows == 8 ? TcShape<64, 1>::kWarps : rows == 16 ? TcShape<64, 2>::kWarps : TcShape<64, 4>::kWarps;
}

cudaError_t launch_decode_tc(const DecodeParams &p, int dtype, cudaStream_t s) {
  return dtype == SB_DTYPE_BF16 ? launch_shape<__nv_bfloat16>(p, s) : launch_shape<__half>(p, s);
}

// 1, 4, 8 or 32 warps share a part, by the chunks that there are for an item, which is about how many pieces it has where it is long
// enough.  The whole call in us with 1, 4, 8, 32, bf16, 128 columns.  1.7 chunks per item (64 sequences x 16 heads): 155, 166, 184, 307;
// 3.8 (29 x 16, 4096 tokens): 162, 167, 177, 240; 4.4 (25 x 16): 141, 145, 154, 208; 9 (12 x 16): 76.6, 76.3, 80, 108; 15 (15 x 8, 8192 tokens):
// 92, 90, 93, 112; 17 (13 x 8): 84, 81, 83, 100; 37 (12 x 4): 52, 46, 45, 53; 111 (1 x 16, 16384 tokens): 55, 39, 34, 35; 222 (1 x 8,
// 32768): 79, 44, 37.5, 34.8; 296 (1 x 6): 94, 45, 35, 31; 444 (1 x 4, 131072): 150, 79, 63, 57.
cudaError_t launch_decode_tc_join(const DecodeParams &p, int dtype, cudaStream_t s) {
  const long long items = (long long)p.batch * p.items_per_seq;
  const int notes = (int)(p.by_item ? items : p.chunks), jobs = p.rows_per_block / 8 * (p.part_cols / 16);
  const int together = p.chunks < 4 * items ? 1 : p.chunks < 16 * items ? 4 : p.chunks < 256 * items ? 8 : 32;
  auto go = [&](auto kernel, int warps, int per_block) {
    return launch_kernel(kernel, dim3(notes, (jobs + per_block - 1) / per_block), warps * 32, 0, s, p);
  };
#define SB_JOIN(T)                                                  \
  together == 32  ? go(decode_tc_join_kernel<T, 32, 32>, 32, 1)     \
  : together == 8 ? go(decode_tc_join_kernel<T, 8, 8>, 8, 1)        \
  : together == 4 ? go(decode_tc_join_kernel<T, 4, 4>, 4, 1)        \
                  : go(decode_tc_join_kernel<T, 4, 1>, 4, 4)
  return dtype == SB_DTYPE_BF16 ? SB_JOIN(__nv_bfloat16) : SB_JOIN(__half);
#undef SB_JOIN
}

}  // namespace sb
