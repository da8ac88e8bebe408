// gated.cu -- the gated feed-forward block and its backward pass.
//
//   forward   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u
//   backward  dg = dh * u * act'(g),  du = dh * act(g)
//             dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg, dbu = column sums
//
// 16-bit types run on the tensor cores: the forward is one launch of the gated tile kernel
// (both projections, the biases, the activation and the product); the backward is one
// elementwise pass (dg, du and the bias sums' partials), one launch for dx whose K axis runs
// over dg Wg and then du Wu in the same accumulator, and one launch for both weight gradients.
// dg and du are rounded to the operands' type once, because the tensor cores read them in it, FP16
// under a common power of two where its range would lose them (fp16_scale);
// the pre-activations that the forward keeps for the backward are FP32, since rounding them
// too would double the rounding error that reaches the gradients.
//
// FP32 runs on the strict FP32 GEMM kernel.  There the product takes 2 k / 3 FMAs per float
// the elementwise passes move: at k = 1024 and more the passes are under 3% of the time, so they
// stay separate kernels.
#include "feed_pair.cuh"
#include "feed_rows.cuh"
#include "feed_split.cuh"
#include "kernels.hpp"

#include <algorithm>
#include <cstddef>

namespace xvram {

using namespace feed;

namespace {

uint64_t up(uint64_t v, uint64_t q) { return (v + q - 1) / q * q; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------------- elementwise passes
// FP32 forward: out = act(g + bg) * (u + bu); with `keep`, g and u are left with their biases.
__global__ void __launch_bounds__(256)
    gate_forward_kernel(float* __restrict__ g, float* __restrict__ u, long long ldg,
                        const float* __restrict__ bg, const float* __restrict__ bu, bool keep,
                        float* __restrict__ out, long long ldo, int rows, int cols, int act) {
  const long long groups = (cols + 3) / 4, total = groups * rows;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / groups;
    const int c = static_cast<int>(i - r * groups) * 4;
    float4* gp = reinterpret_cast<float4*>(g + r * ldg + c);
    float4* wp = reinterpret_cast<float4*>(u + r * ldg + c);
    const float4 g4 = *gp, u4 = *wp;
    float v[4] = {g4.x, g4.y, g4.z, g4.w}, w[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (bg && c + j < cols)
        v[j] += bg[c + j];
      if (bu && c + j < cols)
        w[j] += bu[c + j];
    }
    if (keep && bg)
      *gp = make_float4(v[0], v[1], v[2], v[3]);
    if (keep && bu)
      *wp = make_float4(w[0], w[1], w[2], w[3]);
    gate<false>(act, v, w);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < cols)
        out[r * ldo + c + j] = v[j];
  }
}

constexpr int kBwdRows = 64;  // rows of a block's tile, one partial of the bias sums
constexpr int kBwdCols = 128; // columns of a block's tile, 4 per lane

template <int ACT, bool FAST>
__device__ __forceinline__ void gate_slope(float g, float u, float d, float& dg, float& du) {
  float a, s;
  act_and_slope<ACT, FAST>(g, a, s);
  dg = d * u * s;
  du = d * a;
}

// dg, du (rounded to T) from dh and the kept pre-activations; with `partial`, the tile's FP32
// column sums of the unrounded dg and du, summed in row order.  HBM-bound: 8 bytes of g and u,
// one dh and two results per element.
//
// FP16: `top` receives the largest finite magnitude of dg and du.  `again` is the pass after it: where
// that asks for a scale, dg and du once more times the scale, else nothing.  Clearing `top` and this
// pass cost 4 us of the 68 that the backward of 1021 x 1001 x 2730 takes on the device, 10 us
// where it scales; 8192 x 4096 x 8192 with scaling 6 to 12% more.
template <class T, int ACT>
__global__ void __launch_bounds__(256)
    gate_backward_kernel(const float* __restrict__ g, const float* __restrict__ u, long long ldp,
                         const T* __restrict__ dh, long long lddh, bool vec_dh, T* __restrict__ dg,
                         T* __restrict__ du, long long ldd, float* __restrict__ partial, unsigned* top,
                         bool again, int rows, int cols) {
  constexpr bool kRange = std::is_same_v<T, __half>;
  float scale = 1.0f;
  unsigned most = 0;
  if (kRange && again) {
    scale = fp16_scale(*top);
    if (scale == 1.0f)
      return;
  }
  __shared__ float sums[8][2][kBwdCols];
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * kBwdCols + lane * 4;
  const long long r0 = static_cast<long long>(blockIdx.y) * kBwdRows;
  float sg[4] = {}, su[4] = {};
  for (int k = 0; k < kBwdRows / 8; ++k) {
    const long long r = r0 + k * 8 + ty;
    if (r >= rows || c >= cols)
      continue;
    const float4 g4 = *reinterpret_cast<const float4*>(g + r * ldp + c);
    const float4 u4 = *reinterpret_cast<const float4*>(u + r * ldp + c);
    float d[4] = {};
    if (vec_dh && c + 4 <= cols) {
      if constexpr (sizeof(T) == 2) {
        const uint2 raw = *reinterpret_cast<const uint2*>(dh + r * lddh + c);
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d[j] = to_float(t[j]);
      } else {
        const float4 t = *reinterpret_cast<const float4*>(dh + r * lddh + c);
        d[0] = t.x, d[1] = t.y, d[2] = t.z, d[3] = t.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols)
          d[j] = to_float(dh[r * lddh + c + j]);
    }
    const float gv[4] = {g4.x, g4.y, g4.z, g4.w}, uv[4] = {u4.x, u4.y, u4.z, u4.w};
    alignas(16) T og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // Columns past the end (inside the rows' padding) are written as zeros.
      float a = 0.0f, b = 0.0f;
      if (c + j < cols)
        gate_slope<ACT, sizeof(T) == 2>(gv[j], uv[j], d[j], a, b);
      sg[j] += a;
      su[j] += b;
      if constexpr (kRange) {
        for (float v : {a, b}) {
          const unsigned bits = __float_as_uint(v) & 0x7fffffffu;
          most = max(most, bits < 0x7f800000u ? bits : 0u);
        }
        a *= scale;
        b *= scale;
      }
      og[j] = from_float<T>(a);
      ou[j] = from_float<T>(b);
    }
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(dg + r * ldd + c) = *reinterpret_cast<const uint2*>(og);
      *reinterpret_cast<uint2*>(du + r * ldd + c) = *reinterpret_cast<const uint2*>(ou);
    } else {
      *reinterpret_cast<float4*>(dg + r * ldd + c) = *reinterpret_cast<const float4*>(og);
      *reinterpret_cast<float4*>(du + r * ldd + c) = *reinterpret_cast<const float4*>(ou);
    }
  }
  if (kRange && !again && top) {
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0 && most > *static_cast<volatile unsigned*>(top))
      atomicMax(top, most); // the same bits in any order
  }
  if (!partial)
    return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sums[ty][0][lane * 4 + j] = sg[j];
    sums[ty][1][lane * 4 + j] = su[j];
  }
  __syncthreads();
  const int which = threadIdx.x >> 7, cc = threadIdx.x & 127;
  float t = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    t += sums[k][which][cc];
  const int col = blockIdx.x * kBwdCols + cc;
  if (col < cols)
    partial[(static_cast<long long>(blockIdx.y) * 2 + which) * cols + col] = t;
}

// db[c] = sum of the row tiles' partials, in their order (the same bits every time).
template <class T>
__global__ void __launch_bounds__(256)
    bias_sum_kernel(const float* __restrict__ partial, int tiles, int cols, T* __restrict__ dbg,
                    T* __restrict__ dbu) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= 2ll * cols)
    return;
  T* out = i < cols ? dbg : dbu;
  if (!out)
    return;
  float t = 0.0f;
#pragma unroll 8
  for (int k = 0; k < tiles; ++k)
    t += partial[k * 2ll * cols + i];
  out[i < cols ? i : i - cols] = from_float<T>(t);
}

template <class T>
cudaError_t launch_gate_backward(const GatedProblem& p, const void* dh, long long lddh, T* dg,
                                 T* du, long long ldd, float* partial, unsigned* top, bool again,
                                 cudaStream_t stream) {
  const unsigned tiles_c = (p.h + kBwdCols - 1) / kBwdCols;
  const unsigned tiles_r = (p.m + kBwdRows - 1) / kBwdRows;
  // Row tiles are the grid's y, at most 65535: taller inputs run in slabs.
  const T* d = static_cast<const T*>(dh);
  const bool vec = lddh % 4 == 0 && (reinterpret_cast<uintptr_t>(dh) % (4 * sizeof(T))) == 0;
  for (unsigned t0 = 0; t0 < tiles_r; t0 += 65535) {
    const long long r0 = static_cast<long long>(t0) * kBwdRows;
    const dim3 grid(tiles_c, std::min(tiles_r - t0, 65535u));
    const auto run = [&](auto kernel) {
      kernel<<<grid, 256, 0, stream>>>(p.pre_gate + r0 * p.ld_pre, p.pre_up + r0 * p.ld_pre,
                                       p.ld_pre, d + r0 * lddh, lddh, vec, dg + r0 * ldd,
                                       du + r0 * ldd, ldd,
                                       partial ? partial + 2ll * t0 * p.h : nullptr, top, again,
                                       static_cast<int>(p.m - r0), p.h);
    };
    switch (p.act) {
    case kSilu: run(gate_backward_kernel<T, kSilu>); break;
    case kGelu: run(gate_backward_kernel<T, kGelu>); break;
    case kGeluTanh: run(gate_backward_kernel<T, kGeluTanh>); break;
    case kRelu: run(gate_backward_kernel<T, kRelu>); break;
    default: run(gate_backward_kernel<T, kSigmoid>);
    }
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <class T>
cudaError_t launch_bias_sum(const float* partial, int m, int h, void* dbg, void* dbu,
                            cudaStream_t stream) {
  const long long cols = 2ll * h;
  bias_sum_kernel<T><<<static_cast<unsigned>((cols + 255) / 256), 256, 0, stream>>>(
      partial, (m + kBwdRows - 1) / kBwdRows, h, static_cast<T*>(dbg), static_cast<T*>(dbu));
  return cudaGetLastError();
}

// ---------------------------------------------------------------- 16-bit tiles
// Map of an operand with `rows` rows (the output's axis) and `k` values each: K-major
// ([rows][ld]) or M-/N-major ([k][ld]).
bool operand_map(CUtensorMap* map, bool bf16, const void* base, long long rows, long long k,
                 long long ld, bool mn, uint32_t box_rows = 128) {
  const auto type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return mn ? tc::encode_map(map, type, base, rows, k, ld * 2, 64, 64)
            : tc::encode_map(map, type, base, k, rows, ld * 2, 64, box_rows);
}

Params base_params(bool bf16, int m, int n, int k_tiles, bool a_mn, bool b_mn, int tile_n) {
  Params p{};
  p.m = m;
  p.n = n;
  p.k_tiles = p.k_split = k_tiles;
  p.tiles_n = (n + tile_n - 1) / tile_n;
  p.batches = 1;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.idesc = idesc_f16(bf16, a_mn, b_mn, 256, 256);
  p.timeout_ns = kernel_wait_limit_ns();
  return p;
}

// The pair kernel, with 512-row tiles where their waves cost less: one runs in 1.75 times a
// 256-row tile's time (8192 x 4096 x 8192, seconds of it back to back under the power cap: 824 us
// against 868; 2048 rows, 4 waves against 7: 225 against 222).
template <Epilogue E, class T>
cudaError_t launch_16(const Maps& maps, const Params& p, cudaStream_t stream) {
  const long long pairs = tc::sm_count() / 2, cols = static_cast<long long>(p.batches) * p.tiles_n;
  const long long one = (cols * ((p.m + 255) / 256) + pairs - 1) / pairs;
  const long long two = (cols * ((p.m + 511) / 512) + pairs - 1) / pairs;
  return 1.75 * two < one ? launch_pairs<Kind::f16, E, T, 2>(maps, p, stream)
                          : launch_pairs<Kind::f16, E, T, 1>(maps, p, stream);
}

template <class T>
cudaError_t forward_16(const GatedProblem& q, void* out, long long ldo, cudaStream_t stream) {
  constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
  Maps maps;
  const bool split = q.m <= 128;
  if (!operand_map(&maps.a[0], bf16, q.x, q.m, q.k, q.ldx, q.x_transposed,
                   split ? split_rows(q.m) : 128) ||
      !operand_map(&maps.b[0], bf16, q.w_gate, q.h, q.k, q.ld_gate, q.w_transposed) ||
      !operand_map(&maps.b[1], bf16, q.w_up, q.h, q.k, q.ld_up, q.w_transposed))
    return cudaErrorInvalidValue;
  maps.a[1] = maps.a[0];
  Params p = base_params(bf16, q.m, q.h, (q.k + 63) / 64, q.x_transposed, q.w_transposed, 128);
  p.act = q.act;
  p.bias0 = q.bias_gate;
  p.bias1 = q.bias_up;
  p.out[0] = p.out[1] = out;
  p.ldo = ldo;
  p.unit = store_unit<T>(out, ldo);
  p.save_gate = q.pre_gate;
  p.save_up = q.pre_up;
  p.lds = q.ld_pre;
  if (split) {
    p.idesc = idesc_f16(bf16, p.a_mn, p.b_mn, 128, 256);
    return launch_split<Kind::f16, Epilogue::gated, T>(maps, p, DirectInput{}, false, stream);
  }
  return launch_16<Epilogue::gated, T>(maps, p, stream);
}

template <class T>
cudaError_t backward_16(const GatedProblem& q, const GatedGradients& d, char* ws,
                        cudaStream_t stream) {
  constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
  const long long ldd = static_cast<long long>(up(q.h, 8));
  const uint64_t one = up(static_cast<uint64_t>(q.m) * ldd * 2, 256);
  T* dg = reinterpret_cast<T*>(ws);
  T* du = reinterpret_cast<T*>(ws + one);
  float* partial = d.db_gate || d.db_up ? reinterpret_cast<float*>(ws + 2 * one) : nullptr;
  const bool products = d.dx || d.dw_gate || d.dw_up;
  unsigned* top = nullptr;
  if (!bf16 && products) {
    top = reinterpret_cast<unsigned*>(ws + 2 * one + gated_partial_bytes(q.m, q.h));
    if (cudaError_t e = cudaMemsetAsync(top, 0, sizeof(*top), stream); e != cudaSuccess)
      return e;
  }
  if (cudaError_t e =
          launch_gate_backward<T>(q, d.dh, d.lddh, dg, du, ldd, partial, top, false, stream);
      e != cudaSuccess)
    return e;
  if (top)
    if (cudaError_t e =
            launch_gate_backward<T>(q, d.dh, d.lddh, dg, du, ldd, nullptr, top, true, stream);
        e != cudaSuccess)
      return e;
  if (partial)
    if (cudaError_t e = launch_bias_sum<T>(partial, q.m, q.h, d.db_gate, d.db_up, stream);
        e != cudaSuccess)
      return e;
  if (d.dx) {
    // dx (m x k): A = dg, then du, along h; B = Wg, then Wu, whose rows are the inputs.
    Maps maps;
    const bool b_mn = !q.w_transposed;
    const uint32_t box = split_rows(q.m);
    if (!operand_map(&maps.a[0], bf16, dg, q.m, q.h, ldd, false, box) ||
        !operand_map(&maps.a[1], bf16, du, q.m, q.h, ldd, false, box) ||
        !operand_map(&maps.b[0], bf16, q.w_gate, q.k, q.h, q.ld_gate, b_mn) ||
        !operand_map(&maps.b[1], bf16, q.w_up, q.k, q.h, q.ld_up, b_mn))
      return cudaErrorInvalidValue;
    const int per = (q.h + 63) / 64;
    Params p = base_params(bf16, q.m, q.k, 2 * per, false, b_mn, 256);
    p.k_split = per;
    p.top = top;
    p.out[0] = p.out[1] = d.dx;
    p.ldo = d.lddx;
    p.unit = store_unit<T>(d.dx, d.lddx);
    // K is 2 h, so few tiles take long: split it up to 128 rows, and above where that is
    // estimated to beat the pairs' waves at 0.3 us a stage.
    const long long pairs = tc::sm_count() / 2;
    const long long waves =
        (static_cast<long long>(p.tiles_n) * ((q.m + 255) / 256) + pairs - 1) / pairs;
    Split split;
    cudaError_t e = choose_split<Kind::f16, Epilogue::plain, T>(p, 0, &split);
    if (e != cudaSuccess)
      return e;
    if (q.m <= 128 || split.us < static_cast<double>(waves) * (3.0 + 0.3 * p.k_tiles)) {
      p.idesc = idesc_f16(bf16, p.a_mn, p.b_mn, 128, 256);
      e = launch_split<Kind::f16, Epilogue::plain, T>(maps, p, DirectInput{}, false, stream);
    } else {
      e = launch_16<Epilogue::plain, T>(maps, p, stream);
    }
    if (e != cudaSuccess)
      return e;
  }
  if (d.dw_gate || d.dw_up) {
    // dW (h x k): A = dg or du by batch, stored along h; B = x along its rows.
    Maps maps;
    const bool b_mn = !q.x_transposed;
    const T* first = d.dw_gate ? dg : du;
    if (!operand_map(&maps.a[0], bf16, first, q.h, q.m, ldd, true) ||
        !operand_map(&maps.a[1], bf16, du, q.h, q.m, ldd, true) ||
        !operand_map(&maps.b[0], bf16, q.x, q.k, q.m, q.ldx, b_mn))
      return cudaErrorInvalidValue;
    maps.b[1] = maps.b[0];
    Params p = base_params(bf16, q.h, q.k, (q.m + 63) / 64, true, b_mn, 256);
    p.batches = d.dw_gate && d.dw_up ? 2 : 1;
    p.top = top;
    p.out[0] = d.dw_gate ? d.dw_gate : d.dw_up;
    p.out[1] = d.dw_up;
    p.ldo = d.ld_dw;
    p.unit = std::min(store_unit<T>(p.out[0], d.ld_dw), store_unit<T>(p.out[1], d.ld_dw));
    if (cudaError_t e = launch_16<Epilogue::plain, T>(maps, p, stream);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

// ---------------------------------------------------------------- padded copies
// Rows of unaligned 16- or 32-bit matrices to rows of whole 16 bytes, up to kPackMax matrices in a
// launch.  A thread writes 16 bytes; where the source is only 2-byte aligned it reads the 4-byte
// words around them (each holds a byte of the row, so no word lies outside the allocation).
struct PackParams {
  PackItem item[kPackMax];
  long long first[kPackMax + 1]; // first 16-byte chunk of each matrix
  int count;
};

__global__ void __launch_bounds__(256) pack_rows_kernel(const PackParams p, int size) {
  const long long total = p.first[p.count];
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    int k = 0;
    while (k + 1 < p.count && i >= p.first[k + 1])
      ++k;
    const PackItem& t = p.item[k];
    const long long chunks = (t.cols * size + 15) / 16, j = i - p.first[k];
    const long long r = j / chunks;
    const long long b = (j - r * chunks) * 16; // byte in the row
    const int bytes = static_cast<int>(min(16ll, t.cols * size - b));
    const char* src = static_cast<const char*>(t.src) + r * t.lds * size + b;
    const uint32_t* w =
        reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t{3});
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 2); // bytes
    uint32_t v[5] = {};
#pragma unroll
    for (int q = 0; q < 5; ++q)
      if (4 * q < bytes + shift)
        v[q] = w[q];
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      o[q] = shift ? __funnelshift_r(v[q], v[q + 1], 16) : v[q];
      const int left = bytes - 4 * q; // bytes of this word inside the row
      o[q] &= left >= 4 ? 0xffffffffu : left > 0 ? 0xffffu : 0u;
    }
    *reinterpret_cast<uint4*>(static_cast<char*>(t.dst) + r * t.ldd * size + b) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------- few rows
template <class T>
cudaError_t forward_rows(const GatedProblem& q, void* out, long long ldo, cudaStream_t stream) {
  RowsParams p{};
  p.x = q.x;
  p.w_gate = q.w_gate;
  p.w_up = q.w_up;
  p.ldx = q.ldx;
  p.ld_gate = q.ld_gate;
  p.ld_up = q.ld_up;
  p.bias_gate = q.bias_gate;
  p.bias_up = q.bias_up;
  p.out = out;
  p.ldo = ldo;
  p.save_gate = q.pre_gate;
  p.save_up = q.pre_up;
  p.lds = q.ld_pre;
  p.m = q.m;
  p.h = q.h;
  p.k = q.k;
  p.act = q.act;
  constexpr long long per = 16 / sizeof(T);
  const bool vec = aligned16(q.x) && aligned16(q.w_gate) && aligned16(q.w_up) &&
                   q.ldx % per == 0 && q.ld_gate % per == 0 && q.ld_up % per == 0;
  return vec ? launch_rows<T, static_cast<int>(per)>(p, stream) : launch_rows<T, 1>(p, stream);
}

// Whether the forward runs on the few-rows kernel.  It reads each weight once per 8 rows of x and
// sustains about 20 TFLOP/s of FP32 FMAs; measured against the tile kernels (device time,
// weights larger than L2 rotated):
//   FP32, 4096 inputs, 8192 features: 44 us for 2 rows (6.1 TB/s), 399 for 64, 865 for 128, against
//   549 us for the FFMA kernel, whose waves of 148 128 x 128 tiles take 0.066 us per input whatever
//   m is; 1024 x 2048: 62 us for 128 rows against 136.  4 m h k / 20 TFLOP/s is below the two GEMMs'
//   2 x 0.066 us k waves while m h < 640k waves.
//   BF16: 4096 x 8192 22.6 us for one row, 34 for 4, against the tensor cores' 25.7; 1024 x 2048 3.4 us
//   for one row and 4.5 for 4, against 7.
bool few_rows(const GatedProblem& q) {
  if (q.x_transposed || q.w_transposed)
    return false;
  if (q.type != GatedType::f32)
    return q.m == 1 || (q.m <= 4 && static_cast<long long>(q.h) * q.k <= 1 << 23);
  if (q.m > 512)
    return false;
  const long long tiles = ((q.h + 127ll) / 128) * ((q.m + 127) / 128), sms = tc::sm_count();
  return static_cast<long long>(q.m) * q.h < 640000 * ((tiles + sms - 1) / sms);
}

// ---------------------------------------------------------------- FP32 on the FFMA kernel
// The GEMM is column-major: a row-major (r, c) array is the column-major c x r matrix.
uint64_t sgemm_scratch_fwd(const GatedProblem& q) {
  return sgemm_workspace_bytes(q.w_transposed ? 0 : 1, q.x_transposed ? 1 : 0, q.h, q.m, q.k);
}
uint64_t sgemm_scratch_bwd(const GatedProblem& q) {
  const uint64_t dx = sgemm_workspace_bytes(q.w_transposed ? 1 : 0, 0, q.k, q.m, q.h);
  const uint64_t dw = sgemm_workspace_bytes(q.x_transposed ? 1 : 0, 1, q.k, q.h, q.m);
  return std::max(dx, dw);
}

cudaError_t forward_f32(const GatedProblem& q, float* out, long long ldo, char* ws,
                        cudaStream_t stream) {
  float *g = q.pre_gate, *u = q.pre_up;
  long long ld = q.ld_pre;
  const bool keep = g != nullptr;
  if (!keep) {
    ld = static_cast<long long>(up(q.h, 4));
    const uint64_t one = up(static_cast<uint64_t>(q.m) * ld * 4, 256);
    g = reinterpret_cast<float*>(ws);
    u = reinterpret_cast<float*>(ws + one);
    ws += 2 * one;
  }
  const uint64_t scratch = sgemm_scratch_fwd(q);
  for (int i = 0; i < 2; ++i) {
    // G^T (h x m) = W (h x k) X^T (k x m)
    const cudaError_t e = sgemm_ffma_ws(
        q.w_transposed ? 0 : 1, q.x_transposed ? 1 : 0, q.h, q.m, q.k, 1.0f,
        static_cast<const float*>(i ? q.w_up : q.w_gate), i ? q.ld_up : q.ld_gate,
        static_cast<const float*>(q.x), q.ldx, 0.0f, i ? u : g, ld, scratch ? ws : nullptr, scratch,
        stream);
    if (e != cudaSuccess)
      return e;
  }
  const long long work = (static_cast<long long>(q.h) + 3) / 4 * q.m;
  const long long blocks = std::min<long long>((work + 255) / 256, 16ll * tc::sm_count());
  gate_forward_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
      g, u, ld, static_cast<const float*>(q.bias_gate), static_cast<const float*>(q.bias_up), keep,
      out, ldo, q.m, q.h, q.act);
  return cudaGetLastError();
}

cudaError_t backward_f32(const GatedProblem& q, const GatedGradients& d, char* ws,
                         cudaStream_t stream) {
  const long long ldd = static_cast<long long>(up(q.h, 4));
  const uint64_t one = up(static_cast<uint64_t>(q.m) * ldd * 4, 256);
  float* dg = reinterpret_cast<float*>(ws);
  float* du = reinterpret_cast<float*>(ws + one);
  float* partial = reinterpret_cast<float*>(ws + 2 * one);
  const uint64_t part = gated_partial_bytes(q.m, q.h);
  char* scratch = ws + 2 * one + part;
  const uint64_t scratch_bytes = sgemm_scratch_bwd(q);
  if (!d.db_gate && !d.db_up)
    partial = nullptr;
  if (cudaError_t e = launch_gate_backward<float>(q, d.dh, d.lddh, dg, du, ldd, partial, nullptr, false,
                                                  stream);
      e != cudaSuccess)
    return e;
  if (partial)
    if (cudaError_t e = launch_bias_sum<float>(partial, q.m, q.h, d.db_gate, d.db_up, stream);
        e != cudaSuccess)
      return e;
  for (int i = 0; i < 2; ++i) {
    const float* grad = i ? du : dg;
    if (d.dx) {
      // dX^T (k x m) (+)= W^T (k x h) G^T (h x m)
      const cudaError_t e = sgemm_ffma_ws(
          q.w_transposed ? 1 : 0, 0, q.k, q.m, q.h, 1.0f,
          static_cast<const float*>(i ? q.w_up : q.w_gate), i ? q.ld_up : q.ld_gate, grad, ldd,
          i ? 1.0f : 0.0f, static_cast<float*>(d.dx), d.lddx, scratch_bytes ? scratch : nullptr,
          scratch_bytes, stream);
      if (e != cudaSuccess)
        return e;
    }
    if (void* dw = i ? d.dw_up : d.dw_gate) {
      // dW^T (k x h) = X^T (k x m) G (m x h)
      const cudaError_t e = sgemm_ffma_ws(
          q.x_transposed ? 1 : 0, 1, q.k, q.h, q.m, 1.0f, static_cast<const float*>(q.x), q.ldx,
          grad, ldd, 0.0f, static_cast<float*>(dw), d.ld_dw, scratch_bytes ? scratch : nullptr,
          scratch_bytes, stream);
      if (e != cudaSuccess)
        return e;
    }
  }
  return cudaSuccess;
}

} // namespace

uint64_t gated_partial_bytes(int m, int h) {
  return up(2ull * ((m + kBwdRows - 1) / kBwdRows) * static_cast<uint64_t>(h) * 4, 256);
}

uint64_t gated_workspace_bytes(const GatedProblem& q, bool backward) {
  if (q.m <= 0 || q.h <= 0 || q.k <= 0)
    return 0;
  const uint64_t m = q.m, h = q.h;
  if (!backward && few_rows(q))
    return 0;
  if (q.type == GatedType::f32) {
    const uint64_t pair = 2 * up(m * up(h, 4) * 4, 256);
    return backward ? pair + gated_partial_bytes(q.m, q.h) + sgemm_scratch_bwd(q)
                    : (q.pre_gate ? 0 : pair) + sgemm_scratch_fwd(q);
  }
  const uint64_t range = q.type == GatedType::f16 ? 256 : 0;
  return backward ? 2 * up(m * up(h, 8) * 2, 256) + gated_partial_bytes(q.m, q.h) + range : 0;
}

cudaError_t gated_forward(const GatedProblem& q, void* out, long long ldo, void* workspace,
                          uint64_t workspace_bytes, cudaStream_t stream) {
  const uint64_t need = gated_workspace_bytes(q, false);
  if (workspace_bytes < need || (need && (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return cudaErrorInvalidValue;
  if (few_rows(q)) {
    switch (q.type) {
    case GatedType::f16: return forward_rows<__half>(q, out, ldo, stream);
    case GatedType::bf16: return forward_rows<__nv_bfloat16>(q, out, ldo, stream);
    default: return forward_rows<float>(q, out, ldo, stream);
    }
  }
  switch (q.type) {
  case GatedType::f16: return forward_16<__half>(q, out, ldo, stream);
  case GatedType::bf16: return forward_16<__nv_bfloat16>(q, out, ldo, stream);
  default:
    return forward_f32(q, static_cast<float*>(out), ldo, static_cast<char*>(workspace), stream);
  }
}

cudaError_t gated_backward(const GatedProblem& q, const GatedGradients& d, void* workspace,
                           uint64_t workspace_bytes, cudaStream_t stream) {
  const uint64_t need = gated_workspace_bytes(q, true);
  if (workspace_bytes < need || (need && (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return cudaErrorInvalidValue;
  char* ws = static_cast<char*>(workspace);
  switch (q.type) {
  case GatedType::f16: return backward_16<__half>(q, d, ws, stream);
  case GatedType::bf16: return backward_16<__nv_bfloat16>(q, d, ws, stream);
  default: return backward_f32(q, d, ws, stream);
  }
}

cudaError_t pack_rows(const PackItem* items, int count, int element_size, cudaStream_t stream) {
  if (count < 1 || count > kPackMax || (element_size != 2 && element_size != 4))
    return cudaErrorInvalidValue;
  PackParams p{};
  p.count = count;
  for (int i = 0; i < count; ++i) {
    p.item[i] = items[i];
    p.first[i + 1] = p.first[i] + items[i].rows * ((items[i].cols * element_size + 15) / 16);
  }
  if (p.first[count] == 0)
    return cudaSuccess;
  const long long blocks =
      std::min<long long>((p.first[count] + 255) / 256, 16ll * tc::sm_count());
  pack_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p, element_size);
  return cudaGetLastError();
}

cudaError_t read_and_clear_kernel_error_gated(unsigned int* out, cudaStream_t stream) {
  return read_and_clear_feed_error(out, stream);
}

} // namespace xvram
