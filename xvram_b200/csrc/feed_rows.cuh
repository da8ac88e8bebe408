// feed_rows.cuh -- the gated block for few rows of x: dot products on the FP32 units, each
// weight row read once.
//
// A warp owns HPW outputs' gate and up rows and MR rows of x: its lanes stride over k, keep
// 2 HPW MR sums in registers, and add them up across the warp by a butterfly that halves the
// number of sums a lane holds with every exchange (NV - 1 + log2(32 / NV) shuffles for NV sums
// instead of 5 NV).  Bound by reading the weights from HBM; x comes from L1.
#pragma once

#include "feed_common.cuh"

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

template <class T>
struct Vec16 { // 16 bytes of values
  static constexpr int n = 16 / sizeof(T);
  alignas(16) T v[n];
};

template <class T>
__device__ __forceinline__ void load_stream(const T* p, Vec16<T>& d) {
  uint4 t;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w)
               : "l"(p));
  *reinterpret_cast<uint4*>(d.v) = t;
}

// VEC: values a lane reads at once (16 bytes' worth, or 1 when rows are not 16-byte aligned).
template <class T, int MR, int HPW, int VEC>
__global__ void __launch_bounds__(256) feed_rows_kernel(const RowsParams p) {
  constexpr int NV = 2 * HPW * MR;
  static_assert((NV & (NV - 1)) == 0 && NV <= 32, "sums are a power of two");
  constexpr int UNROLL = VEC == 1 || NV < 16 ? 4 : 2;
  __shared__ float sums[8][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long h0 = (blockIdx.x * 8ll + warp) * HPW;
  const int r0 = blockIdx.y * MR;
  if (h0 >= p.h)
    return; // whole warps
  const T* x = static_cast<const T*>(p.x) + r0 * p.ldx;
  const T *wg[HPW], *wu[HPW];
#pragma unroll
  for (int i = 0; i < HPW; ++i) { // rows past the end repeat the last one
    const long long h = min(h0 + i, static_cast<long long>(p.h) - 1);
    wg[i] = static_cast<const T*>(p.w_gate) + h * p.ld_gate;
    wu[i] = static_cast<const T*>(p.w_up) + h * p.ld_up;
  }
  long long xo[MR];
#pragma unroll
  for (int r = 0; r < MR; ++r)
    xo[r] = min(r, p.m - 1 - r0) * p.ldx;

  float acc[NV] = {}; // [row][output][gate, up]
  const auto step = [&](int k) {
    if constexpr (VEC == 1) {
      float g[HPW], u[HPW];
#pragma unroll
      for (int i = 0; i < HPW; ++i) {
        g[i] = to_float(wg[i][k]);
        u[i] = to_float(wu[i][k]);
      }
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        const float xv = to_float(x[xo[r] + k]);
#pragma unroll
        for (int i = 0; i < HPW; ++i) {
          acc[(r * HPW + i) * 2] = fmaf(xv, g[i], acc[(r * HPW + i) * 2]);
          acc[(r * HPW + i) * 2 + 1] = fmaf(xv, u[i], acc[(r * HPW + i) * 2 + 1]);
        }
      }
    } else {
      Vec16<T> g[HPW], u[HPW];
#pragma unroll
      for (int i = 0; i < HPW; ++i) {
        load_stream(wg[i] + k, g[i]);
        load_stream(wu[i] + k, u[i]);
      }
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        Vec16<T> xv;
        *reinterpret_cast<uint4*>(xv.v) = *reinterpret_cast<const uint4*>(x + xo[r] + k);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float f = to_float(xv.v[j]);
#pragma unroll
          for (int i = 0; i < HPW; ++i) {
            acc[(r * HPW + i) * 2] = fmaf(f, to_float(g[i].v[j]), acc[(r * HPW + i) * 2]);
            acc[(r * HPW + i) * 2 + 1] = fmaf(f, to_float(u[i].v[j]), acc[(r * HPW + i) * 2 + 1]);
          }
        }
      }
    }
  };
  constexpr int kStride = 32 * VEC;
  int k = lane * VEC;
  for (; k + (UNROLL - 1) * kStride + VEC <= p.k; k += UNROLL * kStride) {
#pragma unroll
    for (int j = 0; j < UNROLL; ++j)
      step(k + j * kStride);
  }
  for (; k + VEC <= p.k; k += kStride)
    step(k);
  // 16-byte rows whose length is not whole 16 bytes: the last k % VEC values, one per lane.
  if constexpr (VEC > 1) {
    const int t = p.k / VEC * VEC + lane;
    if (t < p.k) {
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        const float f = to_float(x[xo[r] + t]);
#pragma unroll
        for (int i = 0; i < HPW; ++i) {
          acc[(r * HPW + i) * 2] = fmaf(f, to_float(wg[i][t]), acc[(r * HPW + i) * 2]);
          acc[(r * HPW + i) * 2 + 1] = fmaf(f, to_float(wu[i][t]), acc[(r * HPW + i) * 2 + 1]);
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
  const int mr = p.m >= 5 ? 8 : p.m >= 3 ? 4 : p.m;
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
  case 4: return two ? run(feed_rows_kernel<T, 4, 2, VEC>) : run(feed_rows_kernel<T, 4, 1, VEC>);
  default:
    // 16-bit operands of more rows run on the tensor cores.
    if constexpr (sizeof(T) == 4)
      return two ? run(feed_rows_kernel<T, 8, 2, VEC>) : run(feed_rows_kernel<T, 8, 1, VEC>);
    return cudaErrorInvalidValue;
  }
}

} // namespace xvram::feed
