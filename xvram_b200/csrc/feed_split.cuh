// feed_split.cuh -- the tensor-core kernel of the feed-forward operators for at most 128 rows, and
// for more where CTA pairs would find too few tiles (operands, epilogues and the accumulator's
// columns: feed_common.cuh).
//
// Bound by reading the weights from HBM: a 128 x 256 accumulator takes all rows of A, so each
// weight is read once, and M = 128 MMAs on fewer rows still finish inside the time of the
// loads.  To occupy all SMs when there are few feature tiles, a cluster of p.splits CTAs
// shares a tile and each takes a range of K; the partial sums meet in distributed shared
// memory, where each CTA adds up a share of the columns in rank order (the same bits every
// time) and applies the epilogue.
//
// A's stage holds only ceil(m / 8) * 8 rows: the MMA's other rows read whatever follows in
// shared memory, and those accumulator rows are never looked at.
//
//   warp 0      one lane: TMA loads; weights first, A once the preceding kernel (the
//               quantisation of A, launched with programmatic overlap) is complete;
//   warp 1      one lane: issues the MMAs;
//   warps 2..9  (MXFP4, few rows) quantise the CTA's K range of A into shared memory, in the
//               layout a TMA load would leave, under the first weights' loads;
//               empty the accumulator into shared memory; then all warps reduce and finish.
#pragma once

#include "mxfp4_block.cuh"
#include "split_rule.hpp"

#include <algorithm>

namespace xvram::feed {

// MXFP4: A as the caller's floats, quantised by the kernel (x = 0: A comes from the maps).
constexpr int kDirectRows = 16;
constexpr int kDirectValues = 65536; // rows x values
constexpr int kDirectBytes = 96 * 1024; // shared memory of a CTA's quantised A, at most
struct DirectInput {
  const void* x;
  long long ldx;
  int type; // 0 FP16, 1 BF16, 2 FP32
  int vec;  // 16-byte loads
  int blocks, k;
};

struct SplitParams {
  Params p;
  DirectInput in;
  int splits;      // cluster size
  int stages;      // ring depth
  int a_bytes;     // A's bytes per stage
  int ring;        // offset of the stage ring (behind a quantised A)
};

constexpr int kSplitSmem = 222 * 1024;
constexpr int kSplitRing = kSplitSmem - 2048; // the rest: alignment and barriers
constexpr int kSplitMaxStages = 12;
constexpr int kPitch = 256 + 4; // floats per row of the partial sums

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Blocks [first, last) of rows 0..m of x, two lanes to a block, to the stages' A tiles (codes,
// 128-byte swizzle) and scale tiles; blocks past the end are zeros with scale 127.
template <class X>
__device__ __forceinline__ void quantize_rows(const DirectInput& in, int m, int first, int last,
                                              unsigned char* codes, int a_bytes,
                                              unsigned char* scales, int thread, int threads) {
  constexpr int kEach = 4; // half blocks per thread and turn, loaded before the first is used
  const X* x = static_cast<const X*>(in.x);
  const int width = 2 * (last - first), units = m * width; // width: a multiple of 16
  const unsigned peers = 3u << (threadIdx.x & 30);
  for (int u0 = thread; u0 < units; u0 += kEach * threads) { // whole groups of 16 lanes
    Values16<X> v[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int u = u0 + j * threads, r = u / width, i = u - r * width;
      if (u < units && first + (i >> 1) < in.blocks)
        load16(x + r * in.ldx, static_cast<long long>(first + (i >> 1)) * kBlock + (i & 1) * 16,
               in.k, in.vec != 0, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int u = u0 + j * threads;
      if (u >= units)
        break;
      const int r = u / width, i = u - r * width;
      const int local = i >> 1, sub = i & 1;
      const bool inside = first + local < in.blocks;
      uint32_t top = inside ? top_of(v[j].t) : 0;
      top = max(top, __shfl_xor_sync(peers, top, 1));
      const uint32_t s = inside ? scale_byte(top) : 127u;
      const uint2 code = inside ? codes16(v[j], s) : make_uint2(0, 0);
      const int stage = local >> 3, chunk = local & 7;
      *reinterpret_cast<uint2*>(codes + stage * a_bytes + r * 128 + ((chunk ^ (r & 7)) * 16) +
                                sub * 8) = code;
      if (sub == 0)
        scales[stage * kScaleTile + (chunk >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 +
               (chunk & 3)] = static_cast<unsigned char>(s);
    }
  }
}

template <Kind K, Epilogue E, class T>
__global__ void __launch_bounds__(kThreads, 1)
    feed_split_kernel(const __grid_constant__ Maps maps, const SplitParams q) {
  constexpr int kTileN = E == Epilogue::gated ? 128 : 256;
  constexpr int kElems = K == Kind::f16 ? 64 : 128; // map elements per 128-byte row
  const Params& p = q.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kSplitRing);
  uint64_t* empty = full + kSplitMaxStages;
  uint64_t* acc_full = empty + kSplitMaxStages;
  uint64_t* a_ready = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(a_ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int rank = q.splits > 1 ? static_cast<int>(tc::cluster_rank()) : 0;
  // Row tiles run fastest: those of one weight tile work at the same time.
  const int tile = static_cast<int>(blockIdx.x / q.splits);
  const int m0 = tile % p.tiles_m * 128, n0 = tile / p.tiles_m * kTileN;
  const int rows = min(128, p.m - m0);
  const int k_begin = static_cast<int>(static_cast<long long>(p.k_tiles) * rank / q.splits);
  const int k_end = static_cast<int>(static_cast<long long>(p.k_tiles) * (rank + 1) / q.splits);
  const bool direct = K == Kind::mxf4 && q.in.x;
  const int count = k_end - k_begin, ahead = min(count, q.stages);
  // A stage: A, both parts of B, A's scales, B's scales; a quantised A lies in front of the ring.
  const uint32_t b_off = direct ? 0 : q.a_bytes, scale_off = b_off + 2 * kPart;
  const uint32_t scale_b_off = scale_off + (direct ? 0 : kScaleTile);
  const uint32_t stage_bytes = K == Kind::mxf4 ? scale_b_off + 2 * kScaleTile : scale_off;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(smem), ring = sbase + q.ring;
  const auto load_b = [&](int kt, int s) {
    const uint32_t bar = smem_u32(&full[s]), base = ring + s * stage_bytes;
    const int seg = kt >= p.k_split, k0 = (kt - (seg ? p.k_split : 0)) * kElems;
    mbar_arrive_expect_tx(&full[s], stage_bytes);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const CUtensorMap* mb = &maps.b[E == Epilogue::gated ? j : seg];
      const int row = E == Epilogue::gated ? n0 : n0 + 128 * j;
      const uint32_t d = base + b_off + j * kPart;
      if (K == Kind::f16 && p.b_mn) {
        tc::tma_load<1>(d, mb, bar, row, k0);
        tc::tma_load<1>(d + kPart / 2, mb, bar, row + 64, k0);
      } else {
        tc::tma_load<1>(d, mb, bar, k0, row);
      }
      if constexpr (K == Kind::mxf4)
        tc::tma_load<1>(base + scale_b_off + kScaleTile * j,
                        &maps.scale_b[E == Epilogue::gated ? j : 0], bar, kt * 256,
                        row / 128);
    }
  };
  const auto load_a = [&](int kt, int s) {
    const uint32_t bar = smem_u32(&full[s]), base = ring + s * stage_bytes;
    const int seg = kt >= p.k_split, k0 = (kt - (seg ? p.k_split : 0)) * kElems;
    if (K == Kind::f16 && p.a_mn) {
      tc::tma_load<1>(base, &maps.a[seg], bar, m0, k0);
      tc::tma_load<1>(base + kPart / 2, &maps.a[seg], bar, m0 + 64, k0);
    } else {
      tc::tma_load<1>(base, &maps.a[seg], bar, k0, m0);
    }
    if constexpr (K == Kind::mxf4)
      tc::tma_load<1>(base + scale_off, &maps.scale_a, bar, kt * 256, m0 / 128);
  };
  if (tid == 0) {
    for (int s = 0; s < q.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(a_ready, 8); // the quantising warps
    *abort_flag = 0;
    fence_mbarrier_init();
    // The producer's own barriers are ready: the first weights need not wait for the rest.
    for (int i = 0; i < ahead; ++i)
      load_b(k_begin + i, i);
  }
  if (warp == 1)
    tc::tmem_alloc<1>(tmem_slot, kTmemCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      if (!direct) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int i = 0; i < ahead; ++i)
          load_a(k_begin + i, i);
      }
      int issued = ahead, s = 0;
      uint32_t phase = 0;
      for (; issued < count; ++issued) {
        if (*abort_flag || !mbar_wait_bounded(&empty[s], phase, p.timeout_ns)) {
          atomicOr(&feed_error, 2u);
          *abort_flag = 1;
          break;
        }
        load_b(k_begin + issued, s);
        if (!direct)
          load_a(k_begin + issued, s);
        if (++s == q.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      // Drain: every stage filled here has been consumed (or times out) before exit.
      for (int i = max(0, issued - q.stages); i < issued; ++i) {
        if (!mbar_wait_bounded(&empty[i % q.stages], (i / q.stages) & 1, p.timeout_ns)) {
          atomicOr(&feed_error, 4u);
          break;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 0;
      if (direct && !mbar_wait_bounded(a_ready, 0, p.timeout_ns)) {
        atomicOr(&feed_error, 1u);
        *abort_flag = 1;
      }
      for (int kt = k_begin; kt < k_end; ++kt) {
        if (*abort_flag || !mbar_wait_bounded(&full[s], phase, p.timeout_ns)) {
          atomicOr(&feed_error, 1u);
          *abort_flag = 1;
          break;
        }
        tc::fence_after();
        const uint32_t base = ring + s * stage_bytes;
        const int i = kt - k_begin;
        const uint32_t a = direct ? sbase + i * q.a_bytes : base;
        if constexpr (K == Kind::f16)
          stage_f16<1>(p, tmem, a, base + b_off, i == 0);
        else
          stage_mxf4<1>(p, tmem, a, base + b_off,
                        direct ? sbase + count * q.a_bytes + i * kScaleTile : base + scale_off,
                        base + scale_b_off, tmem + kScaleCol + s * kScaleCols, i == 0);
        tc::mma_commit(smem_u32(&empty[s]));
        if (++s == q.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      tc::mma_commit(smem_u32(acc_full));
    }
    __syncwarp();
  } else {
    // ------------------------------------------- accumulator to shared memory
    if constexpr (K == Kind::mxf4) {
      if (direct) {
        const int first = 8 * k_begin, last = 8 * k_end, thread = tid - 64;
        unsigned char* scales = smem + count * q.a_bytes;
        if (q.in.type == 0)
          quantize_rows<__half>(q.in, p.m, first, last, smem, q.a_bytes, scales, thread, 256);
        else if (q.in.type == 1)
          quantize_rows<__nv_bfloat16>(q.in, p.m, first, last, smem, q.a_bytes, scales, thread,
                                       256);
        else
          quantize_rows<float>(q.in, p.m, first, last, smem, q.a_bytes, scales, thread, 256);
        // The tensor core reads shared memory through the async proxy.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0)
          mbar_arrive(a_ready);
      }
    }
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const bool ok = mbar_wait_bounded(acc_full, 0, p.timeout_ns * 4);
    if (!ok) {
      atomicOr(&feed_error, 8u);
      *abort_flag = 1;
    }
    tc::fence_after();
    if (32 * quad < rows && __all_sync(0xffffffffu, ok && !*abort_flag)) {
      const int row = 32 * quad + lane;
      const uint32_t t_row = tmem + (static_cast<uint32_t>(32 * quad) << 16);
      float* dst = reinterpret_cast<float*>(smem) + row * kPitch;
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t r[2][16];
        tc::tmem_ld16(t_row + 128 * half + c, r[0]);
        tc::tmem_ld16(t_row + 128 * half + c + 16, r[1]);
        tc::tmem_wait_ld();
        if (row < rows) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(dst + 128 * half + c + i) =
                make_uint4(r[i / 16][i % 16], r[i / 16][i % 16 + 1], r[i / 16][i % 16 + 2],
                           r[i / 16][i % 16 + 3]);
        }
        __syncwarp();
      }
    }
    tc::fence_before();
  }

  // Every wait above is bounded, so all warps of all the cluster's CTAs come here.
  __syncthreads();
  if (q.splits > 1)
    tc::cluster_sync();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free<1>(tmem, kTmemCols);
  }
  // ---------------------------------------------------------- reduce and finish
  const int cols = kTileN / q.splits; // a multiple of 16
  const int groups = cols / 4;
  T* out = static_cast<T*>(p.out[0]) + m0 * p.ldo;
  const long long kept = m0 * p.lds;
  float unscale = 1.0f;
  if constexpr (K == Kind::f16 && E == Epilogue::plain && std::is_same_v<T, __half>)
    unscale = fp16_unscale(p.top);
  for (int i = tid; i < rows * groups; i += kThreads) {
    const int r = i / groups, c = rank * cols + (i - r * groups) * 4;
    const int col = n0 + c;
    if (col >= p.n)
      continue;
    float v[4] = {}, w[4] = {};
    for (int s = 0; s < q.splits; ++s) {
      const uint32_t local = sbase + (r * kPitch + c) * 4;
      const uint32_t from = q.splits > 1 ? tc::cluster_addr(local, s) : local;
      const float4 x = load_cluster(from);
      v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
      if constexpr (E == Epilogue::gated) {
        const float4 y = load_cluster(from + 128 * 4);
        w[0] += y.x, w[1] += y.y, w[2] += y.z, w[3] += y.w;
      }
    }
    if constexpr (K == Kind::f16 && E == Epilogue::plain && std::is_same_v<T, __half>) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] *= unscale;
    }
    add_bias<T>(p.bias0, col, p.n, v);
    if constexpr (E == Epilogue::gated) {
      add_bias<T>(p.bias1, col, p.n, w);
      if (p.save_gate) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.n) {
            p.save_gate[kept + r * p.lds + col + j] = v[j];
            p.save_up[kept + r * p.lds + col + j] = w[j];
          }
      }
      gate<sizeof(T) == 2>(p.act, v, w);
    } else if (p.relu) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = act_of<kRelu, true>(v[j]);
    }
    T* dst = out + r * p.ldo + col;
    if (p.unit == 16 && col + 4 <= p.n) {
      alignas(16) T t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t[j] = from_float<T>(v[j]);
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(t);
      else
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(t);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.n)
          dst[j] = from_float<T>(v[j]);
    }
  }
  if (q.splits > 1)
    tc::cluster_sync(); // no CTA leaves while another reads its sums
}

// Rows of A that a stage holds.
inline int split_rows(int m) { return std::min(128, (m + 7) / 8 * 8); }

template <Kind K, Epilogue E, class T>
cudaError_t allow_split() {
  static std::atomic<uint64_t> done{0};
  return tc::allow_smem(feed_split_kernel<K, E, T>, kSplitSmem, done);
}

// The rule's answer for this kernel on the current device (split_rule.hpp).  a_bytes: a quantised
// A's per stage, 0 when A streams.  Clusters of one CTA per SM; each kernel has its own table.
template <Kind K, Epilogue E, class T>
cudaError_t choose_split(const Params& p, int a_bytes, Split* best) {
  constexpr int kTileN = E == Epilogue::gated ? 128 : 256;
  static CapacityTable table;
  const long long tiles =
      static_cast<long long>((p.m + 127) / 128) * ((p.n + kTileN - 1) / kTileN);
  const long long sms = tc::sm_count();
  *best = Split{};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess)
    return e;
  if (cudaError_t e = allow_split<K, E, T>(); e != cudaSuccess) // the capacity query needs it too
    return e;
  const auto capacity = [&](int size, long long* ctas) {
    return table.ctas(dev, size, ctas, [&](int* clusters) {
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = size;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(static_cast<unsigned>(sms / size * size));
      config.blockDim = dim3(kThreads);
      config.dynamicSmemBytes = kSplitSmem;
      config.attrs = &attr;
      config.numAttrs = 1;
      const cudaError_t e =
          cudaOccupancyMaxActiveClusters(clusters, feed_split_kernel<K, E, T>, &config);
      if (e != cudaSuccess)
        cudaGetLastError();
      return static_cast<int>(e);
    });
  };
  return static_cast<cudaError_t>(cheapest_split(
      tiles, p.k_tiles, sms, a_bytes ? a_bytes + static_cast<int>(kScaleTile) : 0, kDirectBytes,
      capacity, best));
}

// `after`: launched behind a kernel of the same stream that allows programmatic overlap.
template <Kind K, Epilogue E, class T>
cudaError_t launch_split(const Maps& maps, const Params& p, const DirectInput& in, bool after,
                         cudaStream_t stream) {
  constexpr int kTileN = E == Epilogue::gated ? 128 : 256;
  const auto kernel = feed_split_kernel<K, E, T>;
  if (cudaError_t e = allow_split<K, E, T>(); e != cudaSuccess)
    return e;
  SplitParams q;
  q.p = p;
  q.in = in;
  const bool direct = in.x != nullptr;
  q.a_bytes = K == Kind::f16 && p.a_mn ? kPart : split_rows(p.m) * 128;
  q.p.tiles_m = (p.m + 127) / 128;
  Split split;
  if (cudaError_t e = choose_split<K, E, T>(p, direct ? q.a_bytes : 0, &split); e != cudaSuccess)
    return e;
  q.splits = split.splits;
  if (q.splits == 0)
    return cudaErrorNotSupported; // this device's clusters are too small for the quantised rows
  const int most = (p.k_tiles + q.splits - 1) / q.splits; // stages of a CTA
  q.ring = direct ? most * (q.a_bytes + static_cast<int>(kScaleTile)) : 0;
  const int stage = (direct ? 0 : q.a_bytes) + 2 * kPart +
                    (K == Kind::mxf4 ? (direct ? 2 : 3) * kScaleTile : 0);
  q.stages = std::min(K == Kind::mxf4 ? 10 : kSplitMaxStages, (kSplitRing - q.ring) / stage);
  const long long grid =
      static_cast<long long>(q.p.tiles_m) * ((p.n + kTileN - 1) / kTileN) * q.splits;
  if (grid > 0x7fffffffll)
    return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(grid));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSplitSmem;
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  unsigned n = 0;
  if (q.splits > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = q.splits;
    attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  if (after) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  config.attrs = attrs;
  config.numAttrs = n;
  return cudaLaunchKernelEx(&config, kernel, maps, q);
}

} // namespace xvram::feed
