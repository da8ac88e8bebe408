// feed_rows.cuh -- the gated block for few rows of x: dot products on the FP32 units, each
// weight row read once.
//
// A warp owns HPW outputs' gate and up rows and MR rows of x: its lanes stride over k, keep
// 2 HPW MR sums in registers, and add them up across the warp by a butterfly that halves the
// number of sums a lane holds with every exchange (NV - 1 + log2(32 / NV) shuffles for NV sums
// instead of 5 NV).  Bound by reading the weights from HBM; x comes from L1.
#pragma once

#include "feed_common.cuh"

#include <type_traits>

namespace xvram::feed {

struct RowsParams {
  const void *x, *w_gate, *w_up;
  long long ldx, ld_gate, ld_up;
  const void *bias_gate, *bias_up;
  void* out;
  long long ldo;
  float *save_gate, *save_up;
  long long lds;
  int m, h, k, act;
};

template <class T, int N>
struct Values {
  alignas(N * sizeof(T)) T v[N];
};

// Weights: read once, so not kept in L1.  Volatile, so that a block's loads stay together ahead of
// the arithmetic.
template <class T, int N>
__device__ __forceinline__ void load_stream(const T* p, Values<T, N>& d) {
  if constexpr (N * sizeof(T) == 16) {
    uint4 t;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w)
                 : "l"(p));
    *reinterpret_cast<uint4*>(d.v) = t;
  } else if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(d.v[0]) : "l"(p));
  } else {
    unsigned short t;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(t) : "l"(p));
    *reinterpret_cast<unsigned short*>(d.v) = t;
  }
}

// VEC: values a lane reads at once (16 bytes' worth, or 1 when rows are not 16-byte aligned).
template <class T, int MR, int HPW, int VEC>
__global__ void __launch_bounds__(256, 2) feed_rows_kernel(const RowsParams p) {
  constexpr int kSums = 2 * HPW * MR; // and zeros up to a power of two, for the butterfly
  constexpr int NV = kSums <= 2 ? 2 : kSums <= 4 ? 4 : kSums <= 8 ? 8 : kSums <= 16 ? 16 : 32;
  static_assert(kSums <= NV, "at most 32 sums");
  constexpr int UNROLL = VEC > 1 ? 4 : NV > 2 ? 8 : 6;
  __shared__ float sums[8][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long h0 = (blockIdx.x * 8ll + warp) * HPW;
  const int r0 = blockIdx.y * MR;
  if (h0 >= p.h)
    return; // whole warps
  const T *x[MR], *wg[HPW], *wu[HPW];
#pragma unroll
  for (int i = 0; i < HPW; ++i) { // rows past the end repeat the last one
    const long long h = min(h0 + i, static_cast<long long>(p.h) - 1);
    wg[i] = static_cast<const T*>(p.w_gate) + h * p.ld_gate + lane * VEC;
    wu[i] = static_cast<const T*>(p.w_up) + h * p.ld_up + lane * VEC;
  }
#pragma unroll
  for (int r = 0; r < MR; ++r)
    x[r] = static_cast<const T*>(p.x) + min(r0 + r, p.m - 1) * p.ldx + lane * VEC;

  float acc[NV] = {}; // [row][output][gate, up]
  const auto block = [&](auto count) { // `count` steps from the pointers on
    constexpr int U = decltype(count)::value;
    Values<T, VEC> g[U][HPW], u[U][HPW];
#pragma unroll
    for (int j = 0; j < U; ++j) {
#pragma unroll
      for (int i = 0; i < HPW; ++i) {
        load_stream(wg[i] + j * 32 * VEC, g[j][i]);
        load_stream(wu[i] + j * 32 * VEC, u[j][i]);
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        const Values<T, VEC> xv =
            *reinterpret_cast<const Values<T, VEC>*>(x[r] + j * 32 * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float f = to_float(xv.v[e]);
#pragma unroll
          for (int i = 0; i < HPW; ++i) {
            float* a = acc + (r * HPW + i) * 2;
            a[0] = fmaf(f, to_float(g[j][i].v[e]), a[0]);
            a[1] = fmaf(f, to_float(u[j][i].v[e]), a[1]);
          }
        }
      }
    }
  };
  // The pointers advance, so that the loads of an unrolled step differ by constants alone.
  constexpr int kStride = 32 * VEC;
  const auto advance = [&](int by) {
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
      wg[i] += by;
      wu[i] += by;
    }
#pragma unroll
    for (int r = 0; r < MR; ++r)
      x[r] += by;
  };
  int left = p.k - lane * VEC; // values from the pointers to the end
  for (; left >= (UNROLL - 1) * kStride + VEC; left -= UNROLL * kStride) {
    block(std::integral_constant<int, UNROLL>{});
    advance(UNROLL * kStride);
  }
  for (; left >= VEC; left -= kStride) {
    block(std::integral_constant<int, 1>{});
    advance(kStride);
  }
  // 16-byte rows whose length is not whole 16 bytes: the lane whose values end the row.
  if constexpr (VEC > 1) {
    if (left > 0) {
      for (int t = 0; t < left; ++t) {
#pragma unroll
        for (int r = 0; r < MR; ++r) {
          const float f = to_float(x[r][t]);
#pragma unroll
          for (int i = 0; i < HPW; ++i) {
            acc[(r * HPW + i) * 2] = fmaf(f, to_float(wg[i][t]), acc[(r * HPW + i) * 2]);
            acc[(r * HPW + i) * 2 + 1] = fmaf(f, to_float(wu[i][t]), acc[(r * HPW + i) * 2 + 1]);
          }
        }
      }
    }
  }

  // Butterfly: with each exchange a lane keeps the half of its sums that its lane bit names.
  int index = 0;
#pragma unroll
  for (int n = NV, bit = 16; bit; bit >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool high = lane & bit;
      index = index * 2 + (high ? 1 : 0);
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        if (i < n) {
          const float send = high ? acc[i] : acc[i + n], keep = high ? acc[i + n] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
        }
      }
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], bit);
    }
  }
  if ((lane & (32 / NV - 1)) == 0)
    sums[warp][index] = acc[0];
  __syncwarp();
  if (lane < MR * HPW) {
    const int r = r0 + lane / HPW;
    const long long h = h0 + lane % HPW;
    if (r < p.m && h < p.h) {
      float g[1] = {sums[warp][2 * lane]}, u[1] = {sums[warp][2 * lane + 1]};
      if (p.bias_gate)
        g[0] += to_float(static_cast<const T*>(p.bias_gate)[h]);
      if (p.bias_up)
        u[0] += to_float(static_cast<const T*>(p.bias_up)[h]);
      if (p.save_gate) {
        p.save_gate[r * p.lds + h] = g[0];
        p.save_up[r * p.lds + h] = u[0];
      }
      gate<sizeof(T) == 2>(p.act, g, u);
      static_cast<T*>(p.out)[r * p.ldo + h] = from_float<T>(g[0]);
    }
  }
}

// Two outputs per warp halve the reads of x per weight but leave half the warps.  Measured, one
// and two: FP32 4096 x 4096 3 rows 35.2 and 27.3 us, 4096 x 8192 8 rows 70 and 61; BF16
// 4096 x 8192 2 rows 26.2 and 30.8, where x costs less.
template <class T, int VEC>
cudaError_t launch_rows(const RowsParams& p, cudaStream_t stream) {
  const int mr = p.m >= 7 ? 8 : p.m;
  const bool two = mr >= (sizeof(T) == 4 ? 2 : 3) && p.h >= 2 * 8 * tc::sm_count();
  const unsigned per = two ? 16 : 8;
  const dim3 grid((p.h + per - 1) / per, (p.m + mr - 1) / mr);
  if (grid.y > 65535)
    return cudaErrorInvalidConfiguration;
  const auto run = [&](auto kernel) {
    kernel<<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
  };
  switch (mr) {
  case 1: return run(feed_rows_kernel<T, 1, 1, VEC>);
  case 2: return two ? run(feed_rows_kernel<T, 2, 2, VEC>) : run(feed_rows_kernel<T, 2, 1, VEC>);
  case 3: return two ? run(feed_rows_kernel<T, 3, 2, VEC>) : run(feed_rows_kernel<T, 3, 1, VEC>);
  case 4: return two ? run(feed_rows_kernel<T, 4, 2, VEC>) : run(feed_rows_kernel<T, 4, 1, VEC>);
  default:
    // 16-bit operands of more rows run on the tensor cores.
    if constexpr (sizeof(T) == 4) {
      if (mr == 5)
        return two ? run(feed_rows_kernel<T, 5, 2, VEC>) : run(feed_rows_kernel<T, 5, 1, VEC>);
      if (mr == 6)
        return two ? run(feed_rows_kernel<T, 6, 2, VEC>) : run(feed_rows_kernel<T, 6, 1, VEC>);
      return two ? run(feed_rows_kernel<T, 8, 2, VEC>) : run(feed_rows_kernel<T, 8, 1, VEC>);
    }
    return cudaErrorInvalidValue;
  }
}

} // namespace xvram::feed
