// feed_common.cuh -- what the tensor-core kernels of the feed-forward operators share:
// operand geometry, instruction descriptors, activations and the epilogue.
//
//   D[m, n] = sum_k A[m, k] B[n, k]                       FP32 accumulation in TMEM
//   gated:  out[m, h] = act(D[m, h] + b0[h]) * (D'[m, h] + b1[h]), D from B0 and D' from B1
//   plain:  out[m, n] = D[m, n] (+ b0[n], then ReLU)
//
// Operands are 16-bit floats (kind::f16) or MXFP4 codes with their block scales (kind::mxf4).
// The stage geometry is the same for both: 128 bytes of K per operand row and stage, 128-byte
// swizzle, four MMAs of 32 bytes of K.  16-bit operands may also be stored M-/N-major
// (contiguous along their rows); MXFP4 operands are K-major.  Accumulators have 256 columns
// from two 128-row parts of B: for the gated form the gate's and the up projection's rows of
// the same 128 features, so that each epilogue thread finds both pre-activations of an output in
// its own TMEM lane and the product needs no exchange; for the plain form neighbouring rows.
//
// All waits are bounded: a wait that runs out sets a bit of the kernel error word, the CTA
// stops issuing, frees its TMEM and returns.
#pragma once

#include "tc_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace xvram::feed {

constexpr int kThreads = 320; // producer, MMA, 8 epilogue warps
constexpr uint32_t kPart = 128 * 128;        // bytes of one 128-row operand part of a stage
constexpr uint32_t kScaleTile = 1024;        // bytes of a 128-row part's scales of a stage
constexpr uint32_t kScaleBytes = 3 * kScaleTile; // A's and both B parts'
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

// Operands of up to two products that share an accumulator or a launch, and MXFP4 scales.
struct Maps {
  CUtensorMap a[2], b[2], scale_a, scale_b[2];
};

struct Params {
  int m, n;               // output rows and columns
  int k_tiles, k_split;   // stages in all; stages of the first operand pair (a[0], b[0])
  int tiles_m, tiles_n, batches;
  int a_mn, b_mn;         // 16-bit operands stored M-/N-major
  int act, relu;
  const unsigned* top;    // FP16, plain: A holds its values times fp16_scale(*top); null: as they are
  int unit;               // widest access the output rows allow, in bytes (store_unit)
  uint32_t idesc;
  const void *bias0, *bias1;
  void* out[2];           // by batch
  long long ldo;
  float *save_gate, *save_up;
  long long lds;
  unsigned long long timeout_ns;
};

// FP16's range.  dg and du are FP16 operands of products whose results may fit where they do not, so
// they are held times a power of two when their largest finite magnitude (`top`, a float's bits) is
// above FP16's 65504, or below 2^-8, where FP16's smallest step of 2^-24 would be more than 2^-16 of
// it.  It then lies in [2^14, 2^15), and the products' results are multiplied by the inverse,
// exactly.
__device__ __forceinline__ float fp16_scale(unsigned top) {
  if (top == 0 || (top >= 0x3b800000u && top <= 0x477fe000u)) // 2^-8, 65504
    return 1.0f;
  const int e = min(141 + 127 - static_cast<int>(top >> 23), 227); // 14 - floor(log2 top), at most 100
  return __uint_as_float(static_cast<unsigned>(e) << 23);
}
__device__ __forceinline__ float fp16_unscale(const unsigned* top) {
  return top ? __uint_as_float((254u << 23) - __float_as_uint(fp16_scale(*top))) : 1.0f;
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

template <int PAIR>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (PAIR == 2)
    asm volatile("{\n"
                 "  .reg .pred p;\n"
                 "  setp.ne.b32 p, %6, 0;\n"
                 "  tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, "
                 "%3, [%4], [%5], p;\n"
                 "}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
                 : "memory");
  else
    asm volatile("{\n"
                 "  .reg .pred p;\n"
                 "  setp.ne.b32 p, %6, 0;\n"
                 "  tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, "
                 "%3, [%4], [%5], p;\n"
                 "}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
                 : "memory");
}

// One scale tile (128 rows x 4 blocks, 32 x 16 bytes) from shared memory to 4 TMEM columns,
// replicated over the four lane quarters; for a pair in both CTAs, each from its own shared
// memory.  Unswizzled: 8-row groups are 128 bytes apart.
template <int PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr) {
  const uint64_t desc = static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | (1ull << 16) |
                        (8ull << 32) | (1ull << 46);
  if constexpr (PAIR == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc)
                 : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc)
                 : "memory");
}

// The four MMAs of a 16-bit stage.
template <int PAIR>
__device__ __forceinline__ void stage_f16(const Params& p, uint32_t d, uint32_t a, uint32_t b,
                                          bool first) {
  const uint64_t sa = p.a_mn ? 128 : 2, sb = p.b_mn ? 128 : 2; // 16-byte units per step
  const uint64_t da = p.a_mn ? tc::desc_mnmajor(a) : tc::desc_kmajor(a);
  const uint64_t db = p.b_mn ? tc::desc_mnmajor(b) : tc::desc_kmajor(b);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    tc::mma_f16<PAIR>(d, da + kk * sa, db + kk * sb, p.idesc, (first && kk == 0) ? 0u : 1u);
}

// The scale copies and the four MMAs of an MXFP4 stage.  The scales of a stage have TMEM
// columns of their own, which the stage's next use overwrites only after its MMAs have completed
// (the stage's barrier says so).  K past the end has zero codes and zero (2^-127) scales.
template <int PAIR>
__device__ __forceinline__ void stage_mxf4(const Params& p, uint32_t d, uint32_t a, uint32_t b,
                                           uint32_t scale_a, uint32_t scale_b, uint32_t sf,
                                           bool first) {
  const uint32_t sfa = sf, sfb = sf + 8;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    copy_scales<PAIR>(sfa + 4 * g, scale_a + 512 * g);
    copy_scales<PAIR>(sfb + 8 * g, scale_b + 512 * g);
    copy_scales<PAIR>(sfb + 8 * g + 4, scale_b + kScaleTile + 512 * g);
  }
  const uint64_t da = tc::desc_kmajor(a), db = tc::desc_kmajor(b);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t id = (kk & 1) * 2; // byte of the scale column for this step
    mma_mxf4<PAIR>(d, da + kk * 2, db + kk * 2, p.idesc | (id << 4) | (id << 29),
                   sfa + 4 * (kk >> 1), sfb + 8 * (kk >> 1), (first && kk == 0) ? 0u : 1u);
  }
}

// ---------------------------------------------------------------- activations
// FAST: for results rounded to 16 bits.  __expf(x) is off by up to (2 + 1.173 |x|) 2^-23 relative and
// __fdividef by 2^-22: together below 2^-18 for |x| <= 20 and 2^-16 up to 88, where half a step of the
// types is 2^-11 and 2^-8.  Otherwise the library functions, for FP32 results.
//
// With e = exp(-|v|) and r = 1 / (1 + e), the logistic function q of v and its complement 1 - q are
// r and e r, by v's sign: nothing overflows, and neither comes from a difference, which would leave
// q (1 - q) no digits from v = 17 on.
template <bool FAST>
__device__ __forceinline__ void logistic(float v, float& q, float& complement) {
  const float e = FAST ? __expf(-fabsf(v)) : expf(-fabsf(v));
  const float r = FAST ? __fdividef(1.0f, 1.0f + e) : 1.0f / (1.0f + e);
  const float er = e * r;
  q = v < 0.0f ? er : r; // a NaN stays one
  complement = v < 0.0f ? r : er;
}
// q alone.  FAST, in the tensor cores' epilogues: the direct form, two instructions shorter (MXFP4
// 4096 x 512 x 8192 57 us against 80).  1 + exp(-v) from 2^126 on gives zero, which is off by
// q < 2^-126.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (FAST)
    return __fdividef(1.0f, 1.0f + __expf(-v));
  float q, complement;
  logistic<FAST>(v, q, complement);
  return q;
}
// Phi(v) = erfc(-v / sqrt 2) / 2, the standard normal distribution function, without
// cancellation for v << 0, and e = exp(-v^2 / 2), which its slope needs too.  FAST: with
// z = |v| / sqrt 2, erfc(z) = exp(-z^2) t P(t), t = 1 / (1 + 0.455 z); P is the least-maximum fit of
// degree 7 to exp(z^2) erfc(z) / t over z >= 0 (relative error 8e-7 in FP32, all z).
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float v, float& e) {
  e = FAST ? __expf(-0.5f * v * v) : expf(-0.5f * v * v);
  if constexpr (FAST) {
    const float t = __fdividef(1.0f, fmaf(0.455f * 0.70710678118654752f, fabsf(v), 1.0f));
    float s = 0.06859361380338669f;
    s = fmaf(s, t, -0.238698810338974f);
    s = fmaf(s, t, 0.19744166731834412f);
    s = fmaf(s, t, 0.0389687679708004f);
    s = fmaf(s, t, 0.19179636240005493f);
    s = fmaf(s, t, 0.2283932864665985f);
    s = fmaf(s, t, 0.2568010985851288f);
    s = fmaf(s, t, 0.25670450925827026f);
    const float half = 0.5f * s * t * e;
    return v < 0.0f ? half : 1.0f - half; // a NaN stays one
  } else {
    return 0.5f * erfcf(-v * 0.70710678118654752f);
  }
}

constexpr float kTanhC = 0.79788456080286536f; // sqrt(2 / pi)
constexpr float kTanhK = 0.044715f;

// (1 + tanh(z)) / 2 = sigmoid(2 z), so the tanh form is v * sigmoid(2 c (v + k v^3)), which
// keeps its relative accuracy where tanh is near -1.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == kSilu)
    return v * sigmoid<FAST>(v);
  else if constexpr (ACT == kGelu) {
    float e;
    return v * normal_cdf<FAST>(v, e);
  }
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
    float q, c;
    logistic<FAST>(v, q, c);
    a = v * q;
    d = fmaf(a, c, q);
  } else if constexpr (ACT == kGelu) {
    float e;
    const float q = normal_cdf<FAST>(v, e);
    a = v * q;
    d = fmaf(v * 0.39894228040143268f, e, q);
  } else if constexpr (ACT == kGeluTanh) {
    float q, c;
    logistic<FAST>(2.0f * kTanhC * (v + kTanhK * v * v * v), q, c);
    a = v * q;
    const float t = a * c; // 0 where v^2 below may overflow
    d = t == 0.0f ? q : fmaf(t, 2.0f * kTanhC * fmaf(3.0f * kTanhK * v, v, 1.0f), q);
  } else if constexpr (ACT == kRelu) {
    a = v < 0.0f ? 0.0f : v;
    d = v > 0.0f ? 1.0f : 0.0f;
  } else {
    float c;
    logistic<FAST>(v, a, c);
    d = a * c;
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

// N (whole 16 bytes) values of a row from column `col` on: 16-byte stores when the row allows
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

// ---------------------------------------------------------------- epilogue, by chunks of 16 columns
// Kept in rolled loops: the activations unrolled over a whole row half stalled on instruction
// fetch (9.6k cycles for 64 outputs per thread against 3k).
//
// A warp's 32 rows x 64 bytes of results go through a 2 KB block of shared memory, 16-byte pieces
// swizzled by the row, so that global stores are whole 32-byte sectors.
constexpr int kSubBlock = 32 * 64;
__device__ __forceinline__ unsigned char* sub_piece(unsigned char* block, int row, int piece) {
  return block + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16);
}

// The block's 64 bytes per row to `out`, columns from `col` on.
template <class T>
__device__ __forceinline__ void flush_block(unsigned char* block, T* out, long long ld, int row0,
                                            int col, int m, int n, int unit) {
  constexpr int per = 16 / sizeof(T), width = 64 / sizeof(T);
  const int lane = threadIdx.x & 31;
  __syncwarp();
  if (unit == 16) {
    const int piece = lane & 3, cc = col + piece * per;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      const uint4 raw = *reinterpret_cast<const uint4*>(sub_piece(block, r, piece));
      if (row0 + r < m) {
        T* dst = out + static_cast<long long>(row0 + r) * ld + cc;
        if (cc + per <= n) {
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
  } else {
    // Rows one or two at a time, by 4 bytes or by elements.
    const int rows = min(32, m - row0), left = min(width, n - col);
    const int size = unit == 4 ? 4 : static_cast<int>(sizeof(T)), across = 64 / size;
    const int step = 32 / across > 0 ? 32 / across : 1, first = lane / across;
    const int at = (lane - first * across) * size; // byte in the row
    const int e = at / static_cast<int>(sizeof(T));
#pragma unroll 4
    for (int r = first; r < rows; r += step) {
      T* dst = out + static_cast<long long>(row0 + r) * ld + col + e;
      const unsigned char* src = sub_piece(block, r, at >> 4) + (at & 15);
      if (size == 4 && e + 4 / static_cast<int>(sizeof(T)) <= left)
        *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
      else if (e < left)
        *dst = *reinterpret_cast<const T*>(src);
    }
  }
  __syncwarp();
}

// 16 values as T, and 16-byte pieces of a thread's row to the block from piece `first` on.
template <class T>
struct Packed {
  static constexpr int n = sizeof(T); // 16-byte pieces
  uint4 piece[n];
};
template <class T>
__device__ __forceinline__ Packed<T> pack(const float (&v)[16]) {
  constexpr int per = 16 / sizeof(T);
  Packed<T> r;
#pragma unroll
  for (int i = 0; i < Packed<T>::n; ++i) {
    alignas(16) T t[per];
#pragma unroll
    for (int j = 0; j < per; ++j)
      t[j] = from_float<T>(v[i * per + j]);
    r.piece[i] = *reinterpret_cast<const uint4*>(t);
  }
  return r;
}
template <class T>
__device__ __forceinline__ void put_pieces(unsigned char* block, int first, const Packed<T>& v) {
#pragma unroll
  for (int i = 0; i < Packed<T>::n; ++i)
    *reinterpret_cast<uint4*>(sub_piece(block, threadIdx.x & 31, first + i)) = v.piece[i];
}

// v[i] += bias[col + i], read once per warp.
template <class T>
__device__ __forceinline__ void add_bias_chunk(const void* bias, int col, int n, float (&v)[16]) {
  if (!bias)
    return;
  const int i = threadIdx.x & 15;
  const float b = col + i < n ? to_float(static_cast<const T*>(bias)[col + i]) : 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    v[j] += __shfl_sync(0xffffffffu, b, j);
}

// A warp's share of an accumulator (TMEM lanes of t_row) to results: the gated form's 64 outputs
// or the plain form's 128 columns of column half `half`, of rows row0.. and columns from `col` on.
// `release` is called once the accumulator has been read.  `unscale` is fp16_unscale's for the plain
// form.  Collective over the warp; T is a 16-bit type.
template <Epilogue E, class T, class F>
__device__ __forceinline__ void finish_unit(const Params& p, uint32_t t_row, int half, int row0,
                                            int col, T* out, unsigned char* block, float unscale,
                                            const F& release) {
  static_assert(sizeof(T) == 2, "two chunks fill a block row");
  constexpr int kChunks = E == Epilogue::gated ? 4 : 8;
  const uint32_t base = t_row + half * 16 * kChunks;
  Packed<T> even; // an even chunk's results, until the odd one's complete 64 bytes
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    uint32_t r0[16], r1[16];
    __syncwarp();
    tc::tmem_ld16(base + 16 * c, r0);
    if constexpr (E == Epilogue::gated)
      tc::tmem_ld16(base + 128 + 16 * c, r1);
    tc::tmem_wait_ld();
    const int cc = col + 16 * c;
    const bool last = c == kChunks - 1 || cc + 16 >= p.n || row0 >= p.m;
    if (last)
      release();
    if (cc < p.n && row0 < p.m) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = __uint_as_float(r0[i]);
      if constexpr (E == Epilogue::plain && std::is_same_v<T, __half>) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] *= unscale;
      }
      add_bias_chunk<T>(p.bias0, cc, p.n, v);
      if constexpr (E == Epilogue::gated) {
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = __uint_as_float(r1[i]);
        add_bias_chunk<T>(p.bias1, cc, p.n, w);
        if (p.save_gate) {
          put_pieces<float>(block, 0, pack<float>(v));
          flush_block(block, p.save_gate, p.lds, row0, cc, p.m, p.n, 16);
          put_pieces<float>(block, 0, pack<float>(w));
          flush_block(block, p.save_up, p.lds, row0, cc, p.m, p.n, 16);
        }
        gate<true>(p.act, v, w);
      } else if (p.relu) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = act_of<kRelu, true>(v[i]);
      }
      const Packed<T> now = pack<T>(v);
      if ((c & 1) || last) {
        if (c & 1)
          put_pieces<T>(block, 0, even);
        put_pieces<T>(block, (c & 1) * 2, now);
        flush_block(block, out, p.ldo, row0, col + 16 * (c & ~1), p.m, p.n, p.unit);
      }
      even = now;
    }
    if (last)
      break;
  }
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
// through `block` (shared memory, 16-byte chunks swizzled by the row), then 8 lanes per row
// where rows are 16-byte aligned (unit 16), else one row at a time by 4 bytes or by elements.
constexpr int kStageBlock = 32 * 128;
template <class T, int N>
__device__ __forceinline__ void store_block(unsigned char* block, const float (&v)[N], int from,
                                            T* out, long long ld, int row0, int col, int m, int n,
                                            int unit) {
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
  if (unit == 16) {
    const int c = lane & 7, cc = col + c * per;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (lane >> 3);
      const uint4 raw = *reinterpret_cast<const uint4*>(block + r * 128 + ((c ^ (r & 7)) * 16));
      if (row0 + r < m) {
        T* dst = out + static_cast<long long>(row0 + r) * ld + cc;
        if (cc + per <= n) {
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
  } else {
    const int rows = min(32, m - row0);
    constexpr int pair = 4 / sizeof(T); // elements of 4 bytes
    T* dst = out + static_cast<long long>(row0) * ld + col;
    const int left = n - col;
    if (unit == 4) {
      const int e = lane * pair;
#pragma unroll 4
      for (int r = 0; r < rows; ++r, dst += ld) {
        const uint32_t raw = *reinterpret_cast<const uint32_t*>(
            block + r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4);
        if (e + pair <= left)
          *reinterpret_cast<uint32_t*>(dst + e) = raw;
        else if (e < left)
          dst[e] = *reinterpret_cast<const T*>(&raw);
      }
    } else {
#pragma unroll 4
      for (int r = 0; r < rows; ++r, dst += ld) {
#pragma unroll
        for (int j = 0; j < pair; ++j) {
          const int e = lane + 32 * j, b = e * static_cast<int>(sizeof(T));
          if (e < left)
            dst[e] = *reinterpret_cast<const T*>(block + r * 128 + (((b >> 4) ^ (r & 7)) * 16) +
                                                 (b & 15));
        }
      }
    }
  }
  __syncwarp();
}

// The widest access that every row of `base` allows: 16 bytes, 4, or an element's.
template <class T>
inline int store_unit(const void* base, long long ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(ld * sizeof(T));
  return a % 16 == 0 ? 16 : a % 4 == 0 ? 4 : static_cast<int>(sizeof(T));
}

// v[from + i] += bias[col + i] for i < N: read once per warp, then broadcast from shared memory.
template <class T, int COUNT, int N>
__device__ __forceinline__ void add_bias_rows(unsigned char* block, const void* bias, int col, int n,
                                              float (&v)[N]) {
  if (!bias)
    return;
  const T* b = static_cast<const T*>(bias);
  float* shared = reinterpret_cast<float*>(block);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < COUNT; i += 32)
    shared[i + lane] = col + i + lane < n ? to_float(b[col + i + lane]) : 0.0f;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < COUNT; i += 4) {
    const float4 t = *reinterpret_cast<const float4*>(shared + i);
    v[i] += t.x, v[i + 1] += t.y, v[i + 2] += t.z, v[i + 3] += t.w;
  }
  __syncwarp();
}

// The loaded accumulator half to results: 64 gated or 128 plain columns from `col` on of the
// warp's rows row0.. (the MXFP4 products', which keep no pre-activations).
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
    add_bias_rows<T, 64>(block, p.bias0, col, p.n, g);
    add_bias_rows<T, 64>(block, p.bias1, col, p.n, u);
    gate<sizeof(T) == 2>(p.act, g, u);
#pragma unroll
    for (int i = 0; i < 64; i += kBlockCols)
      store_block(block, g, i, out, p.ldo, row0, col + i, p.m, p.n, p.unit);
  } else {
    add_bias_rows<T, 128>(block, p.bias0, col, p.n, v);
    if (p.relu) {
#pragma unroll
      for (int i = 0; i < 128; ++i)
        v[i] = act_of<kRelu, true>(v[i]);
    }
#pragma unroll
    for (int i = 0; i < 128; i += kBlockCols)
      store_block(block, v, i, out, p.ldo, row0, col + i, p.m, p.n, p.unit);
  }
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
