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
#include "mxfp4_block.cuh"
#include "xvram_b200.h"
#include "kernels.hpp"

#include <algorithm>

namespace xvram {

using namespace feed;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// 2^(s - 127); 255 is NaN and 0 the subnormal 2^-127.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return s == 255 ? __uint_as_float(0x7fc00000u)
                  : __uint_as_float(s ? s << 23 : 0x00400000u);
}

__device__ __forceinline__ size_t scale_index(long long r, int b, int block_tiles) {
  return (static_cast<size_t>(r >> 7) * block_tiles + (b >> 2)) * 512 + (r & 31) * 16 +
         ((r >> 5) & 3) * 4 + (b & 3);
}

// Both passes: blocks of 256 threads as 256 / tx rows of tx threads, `units` threads to a row,
// each for `each` rows: enough bytes in flight per thread that HBM, and not the blocks'
// latency, bounds large matrices, and one row where there are few blocks.
struct PassGrid {
  int tx, each;
  dim3 grid;
};
PassGrid pass_grid(long long rows, int units, int most) {
  PassGrid g;
  g.tx = 8;
  while (g.tx < units && g.tx < 256)
    g.tx *= 2;
  const long long across = (units + g.tx - 1) / g.tx;
  long long per = 256 / g.tx;
  const bool many = across * ((rows + per - 1) / per) >= 16ll * tc::sm_count();
  g.each = many ? most : 1;
  per *= g.each;
  g.grid = dim3(static_cast<unsigned>(across),
                static_cast<unsigned>(std::min((rows + per - 1) / per, 65535ll)));
  return g;
}

// Two lanes to a block, 16 values each: fewer instructions per value than with smaller shares.
// The grid covers the scales' padded rows and blocks, whose bytes it sets to 127.  A product
// launched behind it with programmatic overlap may start loading its weights at once.
constexpr int kQuantizeRows = 2;
template <class T, int EACH>
__global__ void __launch_bounds__(256)
    mxfp4_quantize_kernel(const T* __restrict__ src, long long lds, bool vec, int rows, int cols,
                          int blocks, int block_tiles, unsigned char* __restrict__ codes,
                          unsigned char* __restrict__ scales, int tx) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int unit = blockIdx.x * tx + (threadIdx.x & (tx - 1));
  const int b = unit >> 1, sub = unit & 1, step = 256 / tx;
  const long long padded = (rows + 127ll) / 128 * 128;
  const unsigned peers = 0xffu << (threadIdx.x & 24);
  if (b >= 4 * block_tiles)
    return; // whole groups of 8 lanes
  for (long long r0 = static_cast<long long>(blockIdx.y) * (step * EACH) + threadIdx.x / tx;
       r0 < padded; r0 += static_cast<long long>(gridDim.y) * (step * EACH)) {
    Values16<T> raw[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (r0 + j * step < rows && b < blocks)
        load16(src + (r0 + j * step) * lds, static_cast<long long>(b) * kBlock + sub * 16, cols, vec,
               raw[j]);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const long long r = r0 + j * step;
      const bool inside = r < rows && b < blocks;
      uint32_t top = inside ? top_of(raw[j].t) : 0;
      top = max(top, __shfl_xor_sync(peers, top, 1));
      uint32_t s = scale_byte(top);
      if (inside)
        reinterpret_cast<uint2*>(codes)[(r * blocks + b) * 2 + sub] = codes16(raw[j], s);
      else
        s = 127;
      // Four blocks' scales are neighbouring bytes.
      s |= __shfl_down_sync(peers, s, 2, 8) << 8;
      s |= __shfl_down_sync(peers, s, 4, 8) << 16;
      if ((threadIdx.x & 7) == 0 && r < padded)
        *reinterpret_cast<uint32_t*>(scales + scale_index(r, b, block_tiles)) = s;
    }
  }
}

// 16 bytes of results per thread and row.
constexpr int kDequantizeRows = 8;
template <class T, int EACH>
__global__ void __launch_bounds__(256)
    mxfp4_dequantize_kernel(const unsigned char* __restrict__ codes,
                            const unsigned char* __restrict__ scales, int rows, int cols,
                            int blocks, int block_tiles, T* __restrict__ dst, long long ldd,
                            bool vec, int tx) {
  constexpr int per = 16 / sizeof(T), lanes = kBlock / per; // values per thread, threads per block
  const int unit = blockIdx.x * tx + (threadIdx.x & (tx - 1));
  const int b = unit / lanes, sub = unit % lanes, step = 256 / tx;
  if (b >= blocks)
    return;
  for (long long r0 = static_cast<long long>(blockIdx.y) * (step * EACH) + threadIdx.x / tx;
       r0 < rows; r0 += static_cast<long long>(gridDim.y) * (step * EACH)) {
    uint32_t code[EACH], scale[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const long long r = min(r0 + j * step, rows - 1ll);
      const unsigned char* c = codes + (r * blocks + b) * 16 + sub * (per / 2);
      code[j] = per == 8 ? *reinterpret_cast<const uint32_t*>(c)
                         : *reinterpret_cast<const unsigned short*>(c);
      scale[j] = scales[scale_index(r, b, block_tiles)];
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const long long r = r0 + j * step;
      const float f = scale_value(scale[j]);
      float v[per];
#pragma unroll
      for (int i = 0; i < per; ++i) {
        // The three magnitude bits as the low exponent bits and the top mantissa bit of a
        // float: E2M1 * 2^-126, subnormals included; times 2^126 exactly.
        const uint32_t t = code[j] >> (4 * i);
        v[i] = __uint_as_float(((t & 7u) << 22) | ((t & 8u) << 28)) * 0x1p126f * f;
      }
      if (r < rows)
        store_row(dst + r * ldd, b * kBlock + sub * per, cols, vec, v);
    }
  }
}

template <class T>
bool vec_rows(const void* p, long long ld) {
  return aligned16(p) && ld % static_cast<long long>(16 / sizeof(T)) == 0;
}

template <class T>
cudaError_t quantize(const void* src, long long lds, int rows, int cols, unsigned char* codes,
                     unsigned char* scales, cudaStream_t stream) {
  const int blocks = (cols + kBlock - 1) / kBlock, tiles = (blocks + 3) / 4;
  const PassGrid g = pass_grid((rows + 127ll) / 128 * 128, tiles * 8, kQuantizeRows);
  const auto kernel =
      g.each > 1 ? mxfp4_quantize_kernel<T, kQuantizeRows> : mxfp4_quantize_kernel<T, 1>;
  kernel<<<g.grid, 256, 0, stream>>>(static_cast<const T*>(src), lds, vec_rows<T>(src, lds), rows,
                                     cols, blocks, tiles, codes, scales, g.tx);
  return cudaGetLastError();
}

template <class T>
cudaError_t dequantize(const unsigned char* codes, const unsigned char* scales, int rows, int cols,
                       void* dst, long long ldd, cudaStream_t stream) {
  const int blocks = (cols + kBlock - 1) / kBlock, tiles = (blocks + 3) / 4;
  const PassGrid g =
      pass_grid(rows, blocks * (kBlock * static_cast<int>(sizeof(T)) / 16), kDequantizeRows);
  const auto kernel =
      g.each > 1 ? mxfp4_dequantize_kernel<T, kDequantizeRows> : mxfp4_dequantize_kernel<T, 1>;
  kernel<<<g.grid, 256, 0, stream>>>(codes, scales, rows, cols, blocks, tiles,
                                     static_cast<T*>(dst), ldd, vec_rows<T>(dst, ldd), g.tx);
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

// Few input values can be quantised by the product itself: each CTA brings its K range of them into
// its shared memory while its first weights arrive.  That saves the pass in front, but each
// cluster quantises its rows again, before its first MMA: it pays up to about 16384 values per
// CTA.  Device time of calls in a graph and, in brackets, of calls in a row from Python, direct against
// a pass in front:
//   values per CTA  8192 (4 x 4096 x 8192 gated)    14.0 us (16.5) against 14.3 (16.9)
//                   8192 (1 x 65536 x 1024 linear)  23.6 us (25.8) against 26.6 (28.9)
//                  16384 (8 x 4096 x 8192 gated)    14.9 us (16.6) against 14.3 (16.9)
//                  16384 (16 x 2048 x 8192 gated)   11.6 us (14.2) against 10.7 (17.3)
//                  24576 (12 x 4096 x 8192 gated)   16.0 us (18.6) against 14.1 (16.9)
//                  32768 (16 x 4096 x 8192 gated)   16.9 us (18.6) against 14.1 (16.9)
static_assert(kDirectRows == XVRAM_B200_MXFP4_DIRECT_ROWS &&
                  kDirectValues == XVRAM_B200_MXFP4_DIRECT_VALUES,
              "the header says the same");
constexpr long long kDirectShare = 16384;

template <Epilogue E, class T>
cudaError_t choose_direct(const Mxfp4Product& q, const Params& p, bool* direct) {
  *direct = q.x && q.m <= kDirectRows && static_cast<long long>(q.m) * q.k <= kDirectValues;
  if (!*direct || !q.a.codes) // without memory for the codes there is no choice
    return cudaSuccess;
  Split split;
  if (cudaError_t e = choose_split<Kind::mxf4, E, T>(p, split_rows(q.m) * 128, &split);
      e != cudaSuccess)
    return e;
  *direct = split.splits > 0 &&
            static_cast<long long>(q.m) *
                    std::min<long long>(q.k, (p.k_tiles + split.splits - 1) / split.splits * 256ll) <=
                kDirectShare;
  return cudaSuccess;
}

template <Epilogue E, class T>
cudaError_t product(const Mxfp4Product& q, cudaStream_t stream) {
  constexpr bool gated = E == Epilogue::gated;
  constexpr int kTileN = gated ? 128 : 256;
  const int blocks = (q.k + kBlock - 1) / kBlock;
  const bool split = q.m <= 128;
  Params p{};
  p.m = q.m;
  p.n = q.n;
  p.k_tiles = p.k_split = (blocks + 7) / 8;
  bool direct;
  if (cudaError_t e = choose_direct<E, T>(q, p, &direct); e != cudaSuccess)
    return e;
  const bool after = q.x && !direct;
  if (after)
    if (cudaError_t e = mxfp4_quantize(q.x_type, q.x, q.ldx, q.m, q.k, q.a.codes, q.a.scales, stream);
        e != cudaSuccess)
      return e;
  Maps maps{};
  if (!direct &&
      !operand_maps(&maps.a[0], &maps.scale_a, q.a, q.m, blocks, split ? split_rows(q.m) : 128))
    return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i)
    if (!operand_maps(&maps.b[i], &maps.scale_b[i], q.b[gated ? i : 0], q.n, blocks, 128))
      return cudaErrorInvalidValue;
  maps.a[1] = maps.a[0];
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
  DirectInput x{};
  if (direct) {
    x.x = q.x;
    x.ldx = q.ldx;
    x.type = static_cast<int>(q.x_type);
    x.blocks = blocks;
    x.k = q.k;
    const int size = q.x_type == GatedType::f32 ? 4 : 2;
    x.vec = aligned16(q.x) && q.ldx * size % 16 == 0;
  }
  return split ? launch_split<Kind::mxf4, E, T>(maps, p, x, after, stream)
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
  if (q.b[1].codes) {
    switch (q.type) {
    case GatedType::f16: return product<Epilogue::gated, __half>(q, stream);
    case GatedType::bf16: return product<Epilogue::gated, __nv_bfloat16>(q, stream);
    default: return product<Epilogue::gated, float>(q, stream);
    }
  }
  switch (q.type) {
  case GatedType::f16: return product<Epilogue::plain, __half>(q, stream);
  case GatedType::bf16: return product<Epilogue::plain, __nv_bfloat16>(q, stream);
  default: return product<Epilogue::plain, float>(q, stream);
  }
}

cudaError_t read_and_clear_kernel_error_mxfp4(unsigned int* out, cudaStream_t stream) {
  return read_and_clear_feed_error(out, stream);
}

} // namespace xvram
