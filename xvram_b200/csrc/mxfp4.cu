// mxfp4.cu -- microscaled 4-bit floating point (MXFP4): quantisation, its inverse, and the
// linear and gated products of two MXFP4 operands on the block-scaled tensor-core MMA.
//
//   A block is 32 neighbouring values of a row.  Its scale is X = 2^(s - 127), stored as the
//   byte s (E8M0): s = clamp(floor(log2 max|v|) - 2, -127, 127) + 127, so the largest element
//   lands in [4, 8), the top binade of E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6).  Elements are v / X
//   rounded to nearest even, saturating at 6; dividing by a power of two is exact.  A block that
//   holds a NaN or an infinity gets the NaN scale 255 and reads back as NaN.
//
//   Storage: codes [rows][ceil(cols / 32)][16 bytes], the even element in the low half of its
//   byte; scales in tiles of 128 rows x 4 blocks, 512 bytes each ([row tile][block tile]), byte
//   (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 -- the order in which the tensor core reads them,
//   so a stage's scales arrive by one bulk copy.  Codes past the last column are 0, scales of
//   rows and blocks past the end 127 (1.0), so that padding multiplies to zero.
#include "feed_pair.cuh"
#include "feed_split.cuh"
#include "kernels.hpp"

#include <algorithm>

namespace xvram {

using namespace feed;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kBlock = 32;

// Eight floats to eight E2M1 codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t to_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n"
      "  .reg .b8 b0, b1, b2, b3;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "  cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "  mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// 2^(s - 127); 255 is NaN and 0 the subnormal 2^-127.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return s == 255 ? __uint_as_float(0x7fc00000u)
                  : __uint_as_float(s ? s << 23 : 0x00400000u);
}

// Values v[0..8) from column c of a row; zeros past the end.
template <class T>
__device__ __forceinline__ void load8(const T* row, long long c, int cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    alignas(16) T t[8];
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(row + c);
    } else {
      reinterpret_cast<uint4*>(t)[0] = *reinterpret_cast<const uint4*>(row + c);
      reinterpret_cast<uint4*>(t)[1] = *reinterpret_cast<const uint4*>(row + c + 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = to_float(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = c + i < cols ? to_float(row[c + i]) : 0.0f;
  }
}

__device__ __forceinline__ size_t scale_index(long long r, int b, int block_tiles) {
  return (static_cast<size_t>(r >> 7) * block_tiles + (b >> 2)) * 512 + (r & 31) * 16 +
         ((r >> 5) & 3) * 4 + (b & 3);
}

// Four lanes to a block, eight values each.  HBM-bound: the values in, 17 bytes out per block.
// The grid covers the scales' padded rows and blocks, whose bytes it sets to 127.  A product
// launched behind it with programmatic overlap may start loading its weights at once.
template <class T>
__global__ void __launch_bounds__(256)
    mxfp4_quantize_kernel(const T* __restrict__ src, long long lds, bool vec, int rows, int cols,
                          int blocks, int block_tiles, unsigned char* __restrict__ codes,
                          unsigned char* __restrict__ scales, long long units) {
  asm volatile("griddepcontrol.launch_dependents;");
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < units; i += gridDim.x * 256ll) {
    const int sub = static_cast<int>(i & 3);
    const long long r = (i >> 2) / (4 * block_tiles);
    const int b = static_cast<int>((i >> 2) - r * (4 * block_tiles));
    const bool inside = r < rows && b < blocks;
    float v[8] = {};
    if (inside)
      load8(src + r * lds, static_cast<long long>(b) * kBlock + sub * 8, cols, vec, v);
    // The largest magnitude by its bits, which order NaN above infinity above finite values.
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    const unsigned peers = 0xfu << (threadIdx.x & 28);
    top = max(top, __shfl_xor_sync(peers, top, 1));
    top = max(top, __shfl_xor_sync(peers, top, 2));
    const int e = static_cast<int>(top >> 23); // floor(log2) + 127 of a normal value
    const uint32_t s = e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
    if (inside) {
      uint32_t code = 0;
      if (s != 255) {
        const float inv = __uint_as_float((254u - s) << 23); // 2^(127 - s)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] *= inv;
        code = to_e2m1(v);
      }
      reinterpret_cast<uint32_t*>(codes)[(r * blocks + b) * 4 + sub] = code;
    }
    if (sub == 0)
      scales[scale_index(r, b, block_tiles)] = static_cast<unsigned char>(inside ? s : 127u);
  }
}

template <class T>
__global__ void __launch_bounds__(256)
    mxfp4_dequantize_kernel(const unsigned char* __restrict__ codes,
                            const unsigned char* __restrict__ scales, int cols, int blocks,
                            int block_tiles, T* __restrict__ dst, long long ldd, bool vec,
                            long long units) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < units; i += gridDim.x * 256ll) {
    const int sub = static_cast<int>(i & 3);
    const long long r = (i >> 2) / blocks;
    const int b = static_cast<int>((i >> 2) - r * blocks);
    const uint32_t code = reinterpret_cast<const uint32_t*>(codes)[i];
    const float x = scale_value(scales[scale_index(r, b, block_tiles)]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // The three magnitude bits as the low exponent bits and the top mantissa bit of a float:
      // E2M1 * 2^-126, subnormals included; times 2^126 exactly.
      const uint32_t c = code >> (4 * j);
      v[j] = __uint_as_float(((c & 7u) << 22) | ((c & 8u) << 28)) * 0x1p126f * x;
    }
    store_row(dst + r * ldd, b * kBlock + sub * 8, cols, vec, v);
  }
}

template <class T>
bool vec_rows(const void* p, long long ld) {
  return aligned16(p) && ld % static_cast<long long>(16 / sizeof(T)) == 0;
}

unsigned blocks_for(long long units) {
  return static_cast<unsigned>(
      std::max<long long>(1, std::min<long long>((units + 255) / 256, 16ll * tc::sm_count())));
}

template <class T>
cudaError_t quantize(const void* src, long long lds, int rows, int cols, unsigned char* codes,
                     unsigned char* scales, cudaStream_t stream) {
  const int blocks = (cols + kBlock - 1) / kBlock, tiles = (blocks + 3) / 4;
  const long long units = ((rows + 127ll) / 128 * 128) * tiles * 16ll;
  mxfp4_quantize_kernel<T><<<blocks_for(units), 256, 0, stream>>>(
      static_cast<const T*>(src), lds, vec_rows<T>(src, lds), rows, cols, blocks, tiles, codes,
      scales, units);
  return cudaGetLastError();
}

template <class T>
cudaError_t dequantize(const unsigned char* codes, const unsigned char* scales, int rows, int cols,
                       void* dst, long long ldd, cudaStream_t stream) {
  const int blocks = (cols + kBlock - 1) / kBlock, tiles = (blocks + 3) / 4;
  const long long units = static_cast<long long>(rows) * blocks * 4;
  mxfp4_dequantize_kernel<T><<<blocks_for(units), 256, 0, stream>>>(
      codes, scales, cols, blocks, tiles, static_cast<T*>(dst), ldd, vec_rows<T>(dst, ldd), units);
  return cudaGetLastError();
}

bool operand_maps(CUtensorMap* codes, CUtensorMap* scales, const Mxfp4Operand& o, int rows,
                  int blocks, uint32_t box_rows) {
  const uint64_t pitch = static_cast<uint64_t>(blocks) * 16;
  const uint64_t tiles = (static_cast<uint64_t>(blocks) + 3) / 4;
  return tc::encode_map(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.codes, pitch, rows, pitch, 128,
                        box_rows) &&
         tc::encode_map(scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, o.scales, tiles * 128,
                        (static_cast<uint64_t>(rows) + 127) / 128, tiles * 512, 256, 1, false);
}

template <Epilogue E, class T>
cudaError_t product(const Mxfp4Product& q, bool after, cudaStream_t stream) {
  constexpr bool gated = E == Epilogue::gated;
  constexpr int kTileN = gated ? 128 : 256;
  const int blocks = (q.k + kBlock - 1) / kBlock;
  const bool split = q.m <= 128;
  Maps maps;
  if (!operand_maps(&maps.a[0], &maps.scale_a, q.a, q.m, blocks, split ? split_rows(q.m) : 128))
    return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i)
    if (!operand_maps(&maps.b[i], &maps.scale_b[i], q.b[gated ? i : 0], q.n, blocks, 128))
      return cudaErrorInvalidValue;
  maps.a[1] = maps.a[0];
  Params p{};
  p.m = q.m;
  p.n = q.n;
  p.k_tiles = p.k_split = (blocks + 7) / 8;
  p.tiles_n = (q.n + kTileN - 1) / kTileN;
  p.batches = 1;
  p.act = q.act;
  p.relu = q.relu;
  p.bias0 = q.bias[0];
  p.bias1 = q.bias[1];
  p.out[0] = p.out[1] = q.out;
  p.ldo = q.ldo;
  p.unit = store_unit<T>(q.out, q.ldo);
  p.timeout_ns = kernel_wait_limit_ns();
  p.idesc = idesc_mxf4(split ? 128 : 256, 256);
  return split ? launch_split<Kind::mxf4, E, T>(maps, p, after, stream)
               : launch_pairs<Kind::mxf4, E, T, 1>(maps, p, stream);
}

} // namespace

cudaError_t mxfp4_quantize(GatedType type, const void* src, long long lds, int rows, int cols,
                           unsigned char* codes, unsigned char* scales, cudaStream_t stream) {
  switch (type) {
  case GatedType::f16: return quantize<__half>(src, lds, rows, cols, codes, scales, stream);
  case GatedType::bf16: return quantize<__nv_bfloat16>(src, lds, rows, cols, codes, scales, stream);
  default: return quantize<float>(src, lds, rows, cols, codes, scales, stream);
  }
}

cudaError_t mxfp4_dequantize(GatedType type, const unsigned char* codes,
                             const unsigned char* scales, int rows, int cols, void* dst,
                             long long ldd, cudaStream_t stream) {
  switch (type) {
  case GatedType::f16: return dequantize<__half>(codes, scales, rows, cols, dst, ldd, stream);
  case GatedType::bf16:
    return dequantize<__nv_bfloat16>(codes, scales, rows, cols, dst, ldd, stream);
  default: return dequantize<float>(codes, scales, rows, cols, dst, ldd, stream);
  }
}

cudaError_t mxfp4_product(const Mxfp4Product& q, cudaStream_t stream) {
  const bool after = q.x != nullptr;
  if (after)
    if (cudaError_t e = mxfp4_quantize(q.x_type, q.x, q.ldx, q.m, q.k, q.a.codes, q.a.scales, stream);
        e != cudaSuccess)
      return e;
  if (q.b[1].codes) {
    switch (q.type) {
    case GatedType::f16: return product<Epilogue::gated, __half>(q, after, stream);
    case GatedType::bf16: return product<Epilogue::gated, __nv_bfloat16>(q, after, stream);
    default: return product<Epilogue::gated, float>(q, after, stream);
    }
  }
  switch (q.type) {
  case GatedType::f16: return product<Epilogue::plain, __half>(q, after, stream);
  case GatedType::bf16: return product<Epilogue::plain, __nv_bfloat16>(q, after, stream);
  default: return product<Epilogue::plain, float>(q, after, stream);
  }
}

cudaError_t read_and_clear_kernel_error_mxfp4(unsigned int* out, cudaStream_t stream) {
  return read_and_clear_feed_error(out, stream);
}

} // namespace xvram
