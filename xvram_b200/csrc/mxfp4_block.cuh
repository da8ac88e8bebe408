// mxfp4_block.cuh -- the quantisation of half an MXFP4 block (16 values, two lanes to a block),
// shared by the quantisation pass and by the product that quantises its few input rows itself.
#pragma once

#include "feed_common.cuh"

#include <cuda_fp4.h>

#include <cstring>

namespace xvram::feed {

constexpr int kBlock = 32;

template <class T>
struct Values16 {
  alignas(16) T t[16];
};

// Values from column c of a row on; zeros past the end.
template <class T>
__device__ __forceinline__ void load16(const T* row, long long c, int cols, bool vec,
                                       Values16<T>& v) {
  if (vec && c + 16 <= cols) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i)
      reinterpret_cast<uint4*>(v.t)[i] = reinterpret_cast<const uint4*>(row + c)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v.t[i] = c + i < cols ? row[c + i] : from_float<T>(0.0f);
  }
}

// The largest magnitude (as float bits) by its bits, which order NaN above infinity above finite
// values.
__device__ __forceinline__ uint32_t top_of(const float (&t)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    top = max(top, __float_as_uint(t[i]) & 0x7fffffffu);
  return top;
}
template <class T>
__device__ __forceinline__ uint32_t top_of(const T (&t)[16]) { // two 16-bit values at a time
  const uint32_t* w = reinterpret_cast<const uint32_t*>(t);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    top = __vmaxu2(top, w[i] & 0x7fff7fffu);
  const unsigned short m = static_cast<unsigned short>(max(top >> 16, top & 0xffffu));
  T v;
  memcpy(&v, &m, 2);
  return __float_as_uint(to_float(v));
}

// Eight floats from v[FROM] on to eight E2M1 codes, the first in the lowest four bits.
template <int FROM>
__device__ __forceinline__ uint32_t to_e2m1(const float (&v)[16]) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(
             make_float2(v[FROM + 2 * i], v[FROM + 2 * i + 1]), __NV_E2M1, cudaRoundNearest))
         << (8 * i);
  return r;
}

// The scale byte of a block whose largest magnitude has these bits: floor(log2) - 2, clamped; 255
// when it is a NaN or an infinity.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const int e = static_cast<int>(top >> 23); // floor(log2) + 127 of a normal value
  return e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
}

// 16 values to codes under the scale byte s (255: zeros).
template <class T>
__device__ __forceinline__ uint2 codes16(const Values16<T>& raw, uint32_t s) {
  const float inv = __uint_as_float((254u - min(s, 254u)) << 23); // 2^(127 - s)
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i] = to_float(raw.t[i]) * inv;
  const uint2 code = make_uint2(to_e2m1<0>(v), to_e2m1<8>(v));
  return s == 255 ? make_uint2(0, 0) : code;
}

} // namespace xvram::feed
