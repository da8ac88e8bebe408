// feed_tile.cuh -- the tensor-core tile kernel of the feed-forward operators.
//
//   D[m, n] = sum_k A[m, k] B[n, k]                       FP32 accumulation in TMEM
//   gated:  out[m, h] = act(D[m, h] + b0[h]) * (D'[m, h] + b1[h]), D from B0 and D' from B1
//   plain:  out[m, n] = D[m, n] (+ b0[n], then ReLU)
//
// Operands are 16-bit floats (kind::f16) or MXFP4 codes with their block scales (kind::mxf4).
// The stage geometry is the same for both: 128 bytes of K per operand row and stage, 128-byte
// swizzle, four MMAs of 32 bytes of K.  16-bit operands may also be stored M-/N-major
// (contiguous along their rows); MXFP4 operands are K-major.
//
// One CTA holds 128 rows of A and two 128-row parts of B, so its accumulator is 128 x 256: for the gated
// form part 0 is the gate's weight rows and part 1 the up projection's rows of the same
// features, so each thread of the epilogue finds both pre-activations of an output in its own
// TMEM lane and the product needs no exchange.  The plain form's parts are neighbouring rows
// of one B.
//
//   warp 0      one lane: TMA loads of a stage's operands (and bulk copies of its scales);
//   warp 1      one lane: copies the scales to TMEM, issues the MMAs, commits;
//   warps 2..9  epilogue, two warps per TMEM lane quarter splitting the columns.
//
// All waits are bounded: a wait that runs out sets a bit of the kernel error word, the CTA
// stops issuing, frees its TMEM and returns.
#pragma once

#include "tc_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace xvram::feed {

constexpr int kThreads = 320; // producer, MMA, 8 epilogue warps
constexpr uint32_t kPart = 128 * 128;        // bytes of one 128-row operand part of a stage
constexpr uint32_t kScaleBytes = 3 * 1024;   // A's and both B parts' scales of a stage
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kScaleCol = 256;          // first TMEM column of the MXFP4 scales
constexpr uint32_t kScaleCols = 24;          // per stage: A 2 x 4, B 2 x 8

enum class Kind { f16, mxf4 };
enum class Epilogue { plain, gated };

// Activations, numbered as XVRAM_B200_GATE_*.
enum Act : int { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3, kSigmoid = 4 };

// Sticky error word of this translation unit's kernels: 1 an MMA issuer, 2 a producer, 4 a drain,
// 8 an epilogue gave up waiting.
static __device__ unsigned int feed_error = 0;

struct Maps {
  CUtensorMap a[2], b[2];
};

struct Params {
  int m, n;               // output rows and columns
  int k_tiles, k_split;   // stages in all; stages of the first operand pair (a[0], b[0])
  int last_steps;         // MMA steps of the last stage
  int tiles_m, tiles_n, batches;
  int a_mn, b_mn;         // 16-bit operands stored M-/N-major
  int act, relu;
  int vec_out;            // outputs (and biases) allow 16-byte accesses
  uint32_t idesc;
  // MXFP4: scale tiles of 512 bytes (128 rows x 4 blocks), `scale_k` of them per row tile
  const unsigned char *scale_a, *scale_b[2];
  int scale_k, scale_rows_b;
  const void *bias0, *bias1;
  void* out[2];           // by batch
  long long ldo;
  float *save_gate, *save_up;
  long long lds;
  unsigned long long timeout_ns;
};

template <Kind K>
__host__ __device__ constexpr int stage_bytes() {
  return 3 * kPart + (K == Kind::mxf4 ? kScaleBytes : 0);
}
constexpr int kStages = 4;
template <Kind K>
__host__ __device__ constexpr int smem_bytes() {
  return kStages * stage_bytes<K>() + 1024 + 256;
}

// Instruction descriptors.  16-bit: D F32, operand format (0 FP16, 1 BF16), majors, N and M.
inline uint32_t idesc_f16(bool bf16, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t f = bf16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// MXFP4: E2M1 operands, UE8M0 scales; the scale byte ids are added per MMA.
inline uint32_t idesc_mxf4(int m, int n) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 7) << 27);
}

__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile("{\n"
               "  .reg .pred p;\n"
               "  setp.ne.b32 p, %6, 0;\n"
               "  tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, "
               "[%4], [%5], p;\n"
               "}\n" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
               : "memory");
}

// One scale tile (128 rows x 4 blocks, 32 x 16 bytes) from shared memory to 4 TMEM columns,
// replicated over the four lane quarters.  Unswizzled: 8-row groups are 128 bytes apart.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr) {
  const uint64_t desc = static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | (1ull << 16) |
                        (8ull << 32) | (1ull << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc)
               : "memory");
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, "
               "[%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// ---------------------------------------------------------------- activations
// Fast: for results rounded to 16 bits; __expf and __fdividef are within a few 2^-22 of the
// quotient's value, far below half a step of either type (2^-11, 2^-8).  Otherwise the
// library functions, for FP32 results.
template <bool FAST>
__device__ __forceinline__ float exp_of(float v) {
  return FAST ? __expf(v) : expf(v);
}
template <bool FAST>
__device__ __forceinline__ float sigmoid(float v) {
  // exp(-v) overflows to infinity for very negative v: 1 / inf = 0, as it should be.
  return FAST ? __fdividef(1.0f, 1.0f + __expf(-v)) : 1.0f / (1.0f + expf(-v));
}
// Phi(v), the standard normal distribution function, without cancellation for v << 0.
__device__ __forceinline__ float normal_cdf(float v) { return 0.5f * erfcf(-v * 0.70710678118654752f); }

constexpr float kTanhC = 0.79788456080286536f; // sqrt(2 / pi)
constexpr float kTanhK = 0.044715f;

// (1 + tanh(z)) / 2 = sigmoid(2 z), so the tanh form is v * sigmoid(2 c (v + k v^3)), which
// keeps its relative accuracy where tanh is near -1.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == kSilu)
    return v * sigmoid<FAST>(v);
  else if constexpr (ACT == kGelu)
    return v * normal_cdf(v);
  else if constexpr (ACT == kGeluTanh)
    return v * sigmoid<FAST>(2.0f * kTanhC * (v + kTanhK * v * v * v));
  else if constexpr (ACT == kRelu)
    return v < 0.0f ? 0.0f : v; // NaN passes through
  else
    return sigmoid<FAST>(v);
}

// act(v) and act'(v).
template <int ACT, bool FAST>
__device__ __forceinline__ void act_and_slope(float v, float& a, float& d) {
  if constexpr (ACT == kSilu) {
    const float q = sigmoid<FAST>(v);
    a = v * q;
    d = fmaf(a, 1.0f - q, q);
  } else if constexpr (ACT == kGelu) {
    const float q = normal_cdf(v);
    a = v * q;
    d = fmaf(v * 0.39894228040143268f, exp_of<FAST>(-0.5f * v * v), q);
  } else if constexpr (ACT == kGeluTanh) {
    const float q = sigmoid<FAST>(2.0f * kTanhC * (v + kTanhK * v * v * v));
    a = v * q;
    const float t = a * (1.0f - q); // 0 where v^2 below may overflow
    d = t == 0.0f ? q : fmaf(t, 2.0f * kTanhC * fmaf(3.0f * kTanhK * v, v, 1.0f), q);
  } else if constexpr (ACT == kRelu) {
    a = v < 0.0f ? 0.0f : v;
    d = v > 0.0f ? 1.0f : 0.0f;
  } else {
    a = sigmoid<FAST>(v);
    d = a * (1.0f - a);
  }
}

// g[i] = act(g[i]) * u[i]; the activation is uniform over the launch, so its switch is outside
// the loop.
template <bool FAST, int N>
__device__ __forceinline__ void gate(int act, float (&g)[N], const float (&u)[N]) {
  switch (act) {
  case kSilu:
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = act_of<kSilu, FAST>(g[i]) * u[i];
    break;
  case kGelu:
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = act_of<kGelu, FAST>(g[i]) * u[i];
    break;
  case kGeluTanh:
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = act_of<kGeluTanh, FAST>(g[i]) * u[i];
    break;
  case kRelu:
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = act_of<kRelu, FAST>(g[i]) * u[i];
    break;
  default:
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = act_of<kSigmoid, FAST>(g[i]) * u[i];
  }
}

// ---------------------------------------------------------------- element types
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N (a multiple of 8) values of a row from column `col` on: 16-byte stores when the row allows
// them and all are inside n, else one by one.
template <class T, int N>
__device__ __forceinline__ void store_row(T* row, int col, int n, bool vec, const float (&v)[N]) {
  constexpr int per = 16 / sizeof(T);
  if (vec && col + N <= n) {
#pragma unroll
    for (int i = 0; i < N; i += per) {
      alignas(16) T t[per];
#pragma unroll
      for (int j = 0; j < per; ++j)
        t[j] = from_float<T>(v[i + j]);
      *reinterpret_cast<uint4*>(row + col + i) = *reinterpret_cast<const uint4*>(t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col + i < n)
        row[col + i] = from_float<T>(v[i]);
  }
}

template <class T, int N>
__device__ __forceinline__ void add_bias(const void* bias, int col, int n, float (&v)[N]) {
  if (!bias)
    return;
  const T* b = static_cast<const T*>(bias);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (col + i < n)
      v[i] += to_float(b[col + i]);
}

// 16 output columns from `col` on of this thread's row: TMEM columns c0.. (and 128 + c0.. for the
// up projection) to the result.  Collective over the warp.
template <Epilogue E, class T>
__device__ __forceinline__ void epilogue_chunk(const Params& p, uint32_t t_row, int c0, int col,
                                               int row, T* out) {
  constexpr bool kFast = sizeof(T) == 2;
  if (col >= p.n)
    return; // uniform over the warp
  __syncwarp();
  uint32_t r0[16], r1[16];
  tc::tmem_ld16(t_row + c0, r0);
  if constexpr (E == Epilogue::gated)
    tc::tmem_ld16(t_row + 128 + c0, r1);
  tc::tmem_wait_ld();
  if (row >= p.m)
    return;
  float v[16], w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i] = __uint_as_float(r0[i]);
  add_bias<T>(p.bias0, col, p.n, v);
  if constexpr (E == Epilogue::gated) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w[i] = __uint_as_float(r1[i]);
    add_bias<T>(p.bias1, col, p.n, w);
    if (p.save_gate) {
      store_row(p.save_gate + static_cast<long long>(row) * p.lds, col, p.n, true, v);
      store_row(p.save_up + static_cast<long long>(row) * p.lds, col, p.n, true, w);
    }
    gate<kFast>(p.act, v, w);
  } else if (p.relu) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] = act_of<kRelu, kFast>(v[i]);
  }
  store_row(out, col, p.n, p.vec_out != 0, v);
}

// A warp's half of an accumulator to registers: the gated form's 64 gate and 64 up columns, or the
// plain form's 128 columns.  Collective over the warp.
template <Epilogue E>
__device__ __forceinline__ void load_accumulator(uint32_t t_row, int half, float (&v)[128]) {
  uint32_t r[128 / 16][16];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = E == Epilogue::gated ? (i < 4 ? 64 * half + 16 * i : 128 + 64 * half + 16 * (i - 4))
                                       : 128 * half + 16 * i;
    tc::tmem_ld16(t_row + c, r[i]);
  }
  tc::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 128; ++i)
    v[i] = __uint_as_float(r[i / 16][i % 16]);
}

// A warp's 32 rows x 128 bytes of results, row per lane, to global memory in whole lines:
// through `block` (shared memory, 16-byte chunks swizzled by the row), then 8 lanes per row.
constexpr int kStageBlock = 32 * 128;
template <class T, int N>
__device__ __forceinline__ void store_block(unsigned char* block, const float (&v)[N], int from,
                                            T* out, long long ld, int row0, int col, int m, int n,
                                            bool vec) {
  constexpr int per = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    alignas(16) T t[per];
#pragma unroll
    for (int j = 0; j < per; ++j)
      t[j] = from_float<T>(v[from + c * per + j]);
    *reinterpret_cast<uint4*>(block + lane * 128 + ((c ^ (lane & 7)) * 16)) =
        *reinterpret_cast<const uint4*>(t);
  }
  __syncwarp();
  const int c = lane & 7, cc = col + c * per;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    const uint4 raw = *reinterpret_cast<const uint4*>(block + r * 128 + ((c ^ (r & 7)) * 16));
    if (row0 + r < m) {
      T* dst = out + static_cast<long long>(row0 + r) * ld + cc;
      if (vec && cc + per <= n) {
        *reinterpret_cast<uint4*>(dst) = raw;
      } else {
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < per; ++j)
          if (cc + j < n)
            dst[j] = t[j];
      }
    }
  }
  __syncwarp();
}

// The loaded accumulator half to results: 64 gated or 128 plain columns from `col` on of the
// warp's rows row0...
template <Epilogue E, class T>
__device__ __forceinline__ void finish_rows(const Params& p, float (&v)[128], int row0, int col,
                                            T* out, unsigned char* block) {
  constexpr int kBlockCols = 128 / sizeof(T); // columns of a stored block
  if (col >= p.n || row0 >= p.m)
    return; // uniform over the warp
  if constexpr (E == Epilogue::gated) {
    float g[64], u[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      g[i] = v[i];
      u[i] = v[64 + i];
    }
    add_bias<T>(p.bias0, col, p.n, g);
    add_bias<T>(p.bias1, col, p.n, u);
    if (p.save_gate) {
#pragma unroll
      for (int i = 0; i < 64; i += 32) {
        store_block(block, g, i, p.save_gate, p.lds, row0, col + i, p.m, p.n, true);
        store_block(block, u, i, p.save_up, p.lds, row0, col + i, p.m, p.n, true);
      }
    }
    gate<sizeof(T) == 2>(p.act, g, u);
#pragma unroll
    for (int i = 0; i < 64; i += kBlockCols)
      store_block(block, g, i, out, p.ldo, row0, col + i, p.m, p.n, p.vec_out != 0);
  } else {
    add_bias<T>(p.bias0, col, p.n, v);
    if (p.relu) {
#pragma unroll
      for (int i = 0; i < 128; ++i)
        v[i] = act_of<kRelu, true>(v[i]);
    }
#pragma unroll
    for (int i = 0; i < 128; i += kBlockCols)
      store_block(block, v, i, out, p.ldo, row0, col + i, p.m, p.n, p.vec_out != 0);
  }
}

template <Kind K, Epilogue E, class T>
__global__ void __launch_bounds__(kThreads, 1)
    feed_tile_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int kStageBytes = stage_bytes<K>();
  constexpr int kTileN = E == Epilogue::gated ? 128 : 256;
  constexpr int kElems = K == Kind::f16 ? 64 : 128; // map elements per 128-byte row
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // Tiles in groups of 8 row tiles, so a wave of CTAs shares both operands' tiles in L2.
  const int per_batch = p.tiles_m * p.tiles_n;
  const int batch = blockIdx.x / per_batch, tile = blockIdx.x % per_batch;
  const int span = 8 * p.tiles_n, first_m = (tile / span) * 8;
  const int group_m = min(8, p.tiles_m - first_m);
  const int m0 = (first_m + (tile % span) % group_m) * 128;
  const int n0 = ((tile % span) / group_m) * kTileN;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1)
    tc::tmem_alloc<1>(tmem_slot, kTmemCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sbase = smem_u32(smem);

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int issued = 0;
      for (int kt = 0; kt < p.k_tiles; ++kt) {
        const int s = kt % kStages, fill = kt / kStages;
        if (*abort_flag)
          break;
        if (fill > 0 && !mbar_wait_bounded(&empty[s], (fill - 1) & 1, p.timeout_ns)) {
          atomicOr(&feed_error, 2u);
          *abort_flag = 1;
          break;
        }
        const int seg = kt >= p.k_split;
        const CUtensorMap* ma = &maps.a[seg | batch];
        const int k0 = (kt - (seg ? p.k_split : 0)) * kElems;
        const uint32_t bar = smem_u32(&full[s]);
        const uint32_t dst = sbase + s * kStageBytes;
        uint32_t bytes = 3 * kPart;
        int atoms = 2;
        if constexpr (K == Kind::mxf4) {
          atoms = min(2, p.scale_k - 2 * kt);
          bytes += 3 * 512 * atoms;
        }
        mbar_arrive_expect_tx(&full[s], bytes);
        if (K == Kind::f16 && p.a_mn) {
          tc::tma_load<1>(dst, ma, bar, m0, k0);
          tc::tma_load<1>(dst + kPart / 2, ma, bar, m0 + 64, k0);
        } else {
          tc::tma_load<1>(dst, ma, bar, k0, m0);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const CUtensorMap* mb = &maps.b[E == Epilogue::gated ? j : seg];
          const int row = E == Epilogue::gated ? n0 : n0 + 128 * j;
          const uint32_t d = dst + (1 + j) * kPart;
          if (K == Kind::f16 && p.b_mn) {
            tc::tma_load<1>(d, mb, bar, row, k0);
            tc::tma_load<1>(d + kPart / 2, mb, bar, row + 64, k0);
          } else {
            tc::tma_load<1>(d, mb, bar, k0, row);
          }
        }
        if constexpr (K == Kind::mxf4) {
          const uint32_t sc = dst + 3 * kPart;
          bulk_load(sc, p.scale_a + (static_cast<size_t>(m0 / 128) * p.scale_k + 2 * kt) * 512,
                    512 * atoms, bar);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // A plain tile's second part may lie past the last row tile: its columns are not
            // stored, so any scales do.
            const int rt = E == Epilogue::gated ? n0 / 128 : min(n0 / 128 + j, p.scale_rows_b - 1);
            bulk_load(sc + 1024 * (1 + j),
                      p.scale_b[E == Epilogue::gated ? j : 0] +
                          (static_cast<size_t>(rt) * p.scale_k + 2 * kt) * 512,
                      512 * atoms, bar);
          }
        }
        ++issued;
      }
      // Drain: every stage filled here has been consumed (or times out) before exit.
      for (int kt = issued > kStages ? issued - kStages : 0; kt < issued; ++kt) {
        if (!mbar_wait_bounded(&empty[kt % kStages], (kt / kStages) & 1, p.timeout_ns)) {
          atomicOr(&feed_error, 4u);
          break;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      for (int kt = 0; kt < p.k_tiles; ++kt) {
        const int s = kt % kStages;
        if (*abort_flag)
          break;
        if (!mbar_wait_bounded(&full[s], (kt / kStages) & 1, p.timeout_ns)) {
          atomicOr(&feed_error, 1u);
          *abort_flag = 1;
          break;
        }
        tc::fence_after();
        const uint32_t a = sbase + s * kStageBytes, b = a + kPart;
        if constexpr (K == Kind::f16) {
          const uint64_t da = p.a_mn ? tc::desc_mnmajor(a) : tc::desc_kmajor(a);
          const uint64_t db = p.b_mn ? tc::desc_mnmajor(b) : tc::desc_kmajor(b);
          const uint64_t sa = p.a_mn ? 128 : 2, sb = p.b_mn ? 128 : 2; // 16-byte units per step
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc::mma_f16<1>(tmem, da + kk * sa, db + kk * sb, p.idesc, (kt | kk) ? 1u : 0u);
        } else {
          const uint32_t sc = a + 3 * kPart;
          const uint32_t sfa = tmem + kScaleCol + s * kScaleCols, sfb = sfa + 8;
          const int steps = kt == p.k_tiles - 1 ? p.last_steps : 4;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (2 * g < steps) {
              copy_scales(sfa + 4 * g, sc + 512 * g);
              copy_scales(sfb + 8 * g, sc + 1024 + 512 * g);
              copy_scales(sfb + 8 * g + 4, sc + 2048 + 512 * g);
            }
          }
          const uint64_t da = tc::desc_kmajor(a), db = tc::desc_kmajor(b);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t id = (kk & 1) * 2; // byte of the scale column for this step
            if (kk < steps)
              mma_mxf4(tmem, da + kk * 2, db + kk * 2, p.idesc | (id << 4) | (id << 29),
                       sfa + 4 * (kk >> 1), sfb + 8 * (kk >> 1), (kt | kk) ? 1u : 0u);
          }
        }
        tc::mma_commit<1>(smem_u32(&empty[s]));
      }
      tc::mma_commit<1>(smem_u32(acc_full));
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row = m0 + 32 * quad + lane;
    const bool ok = mbar_wait_bounded(acc_full, 0, p.timeout_ns * 4);
    if (!ok) {
      atomicOr(&feed_error, 8u);
      *abort_flag = 1;
    }
    tc::fence_after();
    if (__all_sync(0xffffffffu, ok && !*abort_flag)) {
      const uint32_t t_row = tmem + (static_cast<uint32_t>(32 * quad) << 16);
      T* out = static_cast<T*>(p.out[batch]) + static_cast<long long>(row) * p.ldo;
      for (int c0 = half * (kTileN / 2); c0 < (half + 1) * (kTileN / 2); c0 += 16)
        epilogue_chunk<E, T>(p, t_row, c0, n0 + c0, row, out);
    }
    tc::fence_before();
  }

  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free<1>(tmem, kTmemCols);
  }
}

template <Kind K, Epilogue E, class T>
cudaError_t launch_tiles(const Maps& maps, const Params& p, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const auto kernel = feed_tile_kernel<K, E, T>;
  if (cudaError_t e = tc::allow_smem(kernel, smem_bytes<K>(), done); e != cudaSuccess)
    return e;
  const long long grid = static_cast<long long>(p.batches) * p.tiles_m * p.tiles_n;
  if (grid <= 0 || grid > 0x7fffffffll)
    return cudaErrorInvalidConfiguration;
  kernel<<<static_cast<unsigned>(grid), kThreads, smem_bytes<K>(), stream>>>(maps, p);
  return cudaGetLastError();
}

inline cudaError_t read_and_clear_feed_error(unsigned int* out, cudaStream_t stream) {
  const unsigned int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, feed_error, sizeof(*out), 0,
                                            cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess)
    e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *out == 0)
    return e;
  e = cudaMemcpyToSymbolAsync(feed_error, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream);
  return e == cudaSuccess ? cudaStreamSynchronize(stream) : e;
}

} // namespace xvram::feed
