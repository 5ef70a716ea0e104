// Parts shared by the sandwich norm's forward and backward kernels: a thread's columns of a
// row, sums over warps and CTAs, parameters, the launch.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace tileops {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Several sums over a warp at once: their shuffles are independent of each other.
template <int K>
__device__ __forceinline__ void warp_sums(float (&v)[K]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

template <typename W>
__device__ __forceinline__ float param(const W* p, int64_t i, float otherwise) {
  return p ? Cvt<W>::to_f(p[i]) : otherwise;
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(in ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's packets of a row: packet j is the row's packet threadIdx.x + j kThreads, kV
// elements.  kBytes = 16: rows of whole packets on 16-byte boundaries.  Otherwise
// the last packet may be short, and packets are copied and written by words of
// 4 bytes (rows of whole words) or by elements of 2, which no asynchronous
// copy takes.
template <typename T, int kThreads, int kPackets, int kBytes>
struct Cols {
  static constexpr int kV = 16 / sizeof(T);
  static constexpr bool kWhole = kBytes == 16;
  static __device__ __forceinline__ int first(int j) { return (threadIdx.x + j * kThreads) * kV; }
  // How many elements packet j has (all or none of an aligned row).
  static __device__ __forceinline__ int count(int j, int N) {
    const int left = N - first(j);
    return kWhole ? (left > 0 ? kV : 0) : max(0, min(kV, left));
  }
  static __device__ __forceinline__ void fetch(uint4* slot, const T* row, int j, int N) {
    if constexpr (kWhole) {
      if (first(j) < N) copy16(slot, row + first(j));
    } else if constexpr (kBytes == 4) {
      constexpr int kEach = 4 / sizeof(T);
      const int n = count(j, N);
      if (n > 0)
#pragma unroll
        for (int i = 0; i < 4; ++i)  // a word past the end is zeros, its source not read
          copy4(reinterpret_cast<uint32_t*>(slot) + i,
                row + first(j) + (i * kEach < n ? i * kEach : 0), i * kEach < n);
    } else {
      T e[kV];
      const int n = count(j, N);
#pragma unroll
      for (int i = 0; i < kV; ++i) e[i] = i < n ? row[first(j) + i] : Cvt<T>::from_f(0.0f);
      memcpy(slot, e, 16);
    }
  }
  // Two neighbouring columns at a time: the arithmetic is packed (fma.rn.f32x2 and its kin).
  static constexpr int kP = kV / 2;
  static __device__ __forceinline__ void read(const uint4* slot, float2 (&v)[kP]) {
    const uint4 u = *slot;
    if constexpr (sizeof(T) == 4) {
      v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
      v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = unpack(w[i]);
    }
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    if constexpr (std::is_same_v<T, __half>) {
      __half2 h;
      memcpy(&h, &w, 4);
      return __half22float2(h);
    } else {
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
  }
  static __device__ __forceinline__ uint32_t pack(float2 v) {
    uint32_t w;
    if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __float22half2_rn(v);
      memcpy(&w, &h, 4);
    } else {
      const __nv_bfloat162 h = __float22bfloat162_rn(v);
      memcpy(&w, &h, 4);
    }
    return w;
  }
  // v rounded to T, as it will be read again.
  static __device__ __forceinline__ void round(float2 (&v)[kP]) {
    if constexpr (sizeof(T) == 2)
#pragma unroll
      for (int i = 0; i < kP; ++i) v[i] = unpack(pack(v[i]));
  }
  static __device__ __forceinline__ void write(T* row, int j, int N, const float2 (&v)[kP]) {
    uint4 u;
    if constexpr (sizeof(T) == 4) {
      u = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                     __float_as_uint(v[1].y));
    } else {
      u = make_uint4(pack(v[0]), pack(v[1]), pack(v[2]), pack(v[3]));
    }
    if constexpr (kWhole) {
      st_stream(row + first(j), u);
    } else if constexpr (kBytes == 4) {
      constexpr int kEach = 4 / sizeof(T);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      const int n = count(j, N);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i * kEach < n) __stcs(reinterpret_cast<uint32_t*>(row + first(j)) + i, w[i]);
    } else {
      T e[kV];
      memcpy(e, &u, 16);
      const int n = count(j, N);
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (i < n) row[first(j) + i] = e[i];
    }
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// (v - mean) rstd; RMS takes no mean.  (The difference first: v rstd - mean rstd would cancel
// where the mean is large.)
template <bool kLayer>
__device__ __forceinline__ float2 normed(float2 v, float mean, float rstd) {
  return fmul2(kLayer ? fadd2(v, both(-mean)) : v, both(rstd));
}
__device__ __forceinline__ float total(float2 v) { return v.x + v.y; }

// Rows of CTA c of C: consecutive, so that a CTA meets few gate groups.
__device__ __forceinline__ int first_row(int64_t M, int c, int C) {
  return static_cast<int>(M * c / C);
}

// ---- statistics of a row over a CTA, one barrier ----
// Each warp publishes kSums numbers; after the barrier lane l takes those of warp
// l % kWarps and the sums over warps are butterflies.  Callers alternate two buffers: one is
// written again only after a barrier that every reader of it has passed.
template <int kSums, int kWarps>
struct WarpSums {
  float v[kSums][kWarps];
};

// Sums over the warps of what lane l holds of warp l % kWarps; in every lane.
template <int kWarps, int K>
__device__ __forceinline__ void over_warps(float (&v)[K]) {
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

// Number of row elements that lie in warp w.
template <typename C, int kThreads, int kPackets>
__device__ __forceinline__ float in_warp(int w, int N) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < kPackets; ++j) {
    const int from = (w * 32 + j * kThreads) * C::kV;
    n += max(0, min(32 * C::kV, N - from));
  }
  return static_cast<float>(n);
}

// A thread's sum of a row, and its sum of squares about `mean`.
template <typename C, int kPackets>
__device__ __forceinline__ float sum_of(const float2 (&v)[kPackets][C::kP]) {
  float2 sum = both(0.0f);
#pragma unroll
  for (int j = 0; j < kPackets; ++j)
#pragma unroll
    for (int i = 0; i < C::kP; ++i) sum = fadd2(sum, v[j][i]);  // zeros past the end
  return total(sum);
}
template <typename C, int kPackets>
__device__ __forceinline__ float squares_of(const float2 (&v)[kPackets][C::kP],
                                            const int (&n)[kPackets], bool layer, float mean) {
  float2 sq = both(0.0f);
#pragma unroll
  for (int j = 0; j < kPackets; ++j)
    if (!layer) {
#pragma unroll
      for (int i = 0; i < C::kP; ++i) sq = ffma2(v[j][i], v[j][i], sq);
    } else if (n[j] > 0) {
#pragma unroll
      for (int i = 0; i < C::kP; ++i) {
        float2 d = fadd2(v[j][i], both(-mean));
        if (!C::kWhole && 2 * i >= n[j]) d.x = 0.0f;
        if (!C::kWhole && 2 * i + 1 >= n[j]) d.y = 0.0f;
        sq = ffma2(d, d, sq);
      }
    }
  return total(sq);
}

// Parameters of a thread's columns: `otherwise` where there is no vector p, zero where there
// is no column.  vec: p starts on a 16-byte boundary (and rows are aligned).
template <typename C, typename W, int kPackets>
__device__ __forceinline__ void load_params(float2 (&v)[kPackets][C::kP], const int (&n)[kPackets],
                                            const W* p, float otherwise, bool vec) {
#pragma unroll
  for (int j = 0; j < kPackets; ++j) {
    const int c = C::first(j);
    if (C::kWhole && vec && p) {
      constexpr int kWords = C::kV * sizeof(W) / 16;  // 16-byte words of a packet's parameters
      alignas(16) W e[C::kV];
      if (n[j] > 0) {
#pragma unroll
        for (int q = 0; q < kWords; ++q)
          reinterpret_cast<uint4*>(e)[q] = __ldg(reinterpret_cast<const uint4*>(p + c) + q);
      }
#pragma unroll
      for (int i = 0; i < C::kP; ++i)
        v[j][i] = n[j] > 0 ? make_float2(Cvt<W>::to_f(e[2 * i]), Cvt<W>::to_f(e[2 * i + 1]))
                           : both(0.0f);
    } else {
#pragma unroll
      for (int i = 0; i < C::kP; ++i)
        v[j][i] = make_float2(2 * i < n[j] ? param(p, c + 2 * i, otherwise) : 0.0f,
                              2 * i + 1 < n[j] ? param(p, c + 2 * i + 1, otherwise) : 0.0f);
    }
  }
}
template <typename C, int kPackets>
__device__ __forceinline__ void multiply(float2 (&v)[kPackets][C::kP],
                                         const float2 (&by)[kPackets][C::kP]) {
#pragma unroll
  for (int j = 0; j < kPackets; ++j)
#pragma unroll
    for (int i = 0; i < C::kP; ++i) v[j][i] = fmul2(v[j][i], by[j][i]);
}

// ---- rows too wide for a thread's registers ----
// Passes over the row, which is read again from L1 or L2; kV columns at a time, a 16-byte
// packet where rows allow it.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  __syncthreads();  // `red` may still be read by the previous reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarps ? red[lane] : 0.0f);
}

template <int kV, typename T>
__device__ __forceinline__ void load_cols(const T* p, float (&v)[kV], bool vec = true) {
  constexpr int kSize = kV * static_cast<int>(sizeof(T));
  T e[kV];
  if (kSize % 16 == 0 && vec) {
#pragma unroll
    for (int q = 0; q < kSize / 16; ++q) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[q];
      memcpy(reinterpret_cast<char*>(e) + 16 * q, &u, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) v[i] = Cvt<T>::to_f(e[i]);
}
// kV parameters from p on, `otherwise` where there is no vector.
template <int kV, typename W>
__device__ __forceinline__ void load_vector(const W* p, int64_t at, float otherwise, bool vec,
                                            float (&v)[kV]) {
  if (p) {
    load_cols<kV>(p + at, v, vec);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = otherwise;
  }
}
template <int kV, typename T>
__device__ __forceinline__ void store_cols(T* p, const float (&v)[kV]) {
  T e[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) e[i] = Cvt<T>::from_f(v[i]);
  if constexpr (kV * sizeof(T) == 16) {
    uint4 u;
    memcpy(&u, e, 16);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) p[i] = e[i];
  }
}

// mean and rstd of a row.
template <int kV, typename T>
__device__ __forceinline__ float2 row_stats(const T* row, int64_t N, bool layer, float eps,
                                            float* red) {
  float mean = 0.0f, sq = 0.0f, v[kV];
  const int64_t first = static_cast<int64_t>(threadIdx.x) * kV, step = blockDim.x * kV;
  if (layer) {
    float sum = 0.0f;
    for (int64_t c = first; c < N; c += step) {
      load_cols<kV>(row + c, v);
#pragma unroll
      for (int i = 0; i < kV; ++i) sum += v[i];
    }
    mean = block_sum(sum, red) / static_cast<float>(N);
  }
  for (int64_t c = first; c < N; c += step) {
    load_cols<kV>(row + c, v);
#pragma unroll
    for (int i = 0; i < kV; ++i) sq = fmaf(v[i] - mean, v[i] - mean, sq);
  }
  return make_float2(mean, 1.0f / sqrtf(block_sum(sq, red) / static_cast<float>(N) + eps));
}

// ---- launches ----
// Calls f with values of the row type and the parameter type.
template <typename F>
int with_types(int dtype, int affine_dtype, F f) {
  const bool wide = affine_dtype == TILEOPS_DT_F32;
  if (!wide && affine_dtype != dtype) return TILEOPS_EBADDTYPE;
  switch (dtype) {
    case TILEOPS_DT_F32: return f(float(), float());
    case TILEOPS_DT_F16: return wide ? f(__half(), float()) : f(__half(), __half());
    case TILEOPS_DT_BF16:
      return wide ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
    default: return TILEOPS_EBADDTYPE;
  }
}

// Calls f with the widest copy that dense rows of N at these addresses allow.
template <typename T, typename F>
int with_bytes(int64_t N, std::initializer_list<const void*> rows, F f) {
  const int64_t row = N * static_cast<int64_t>(sizeof(T));
  auto all = [&](int bytes) {
    bool ok = row % bytes == 0;
    for (const void* p : rows) ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0;
    return ok;
  };
  if (all(16)) return f(std::integral_constant<int, 16>());
  if constexpr (sizeof(T) == 2) {
    if (!all(4)) return f(std::integral_constant<int, 2>());
  }
  return f(std::integral_constant<int, 4>());
}

inline bool bad_shape(int64_t M, int64_t N, int64_t G) {
  return M < 0 || N <= 0 || G < 1 || M > 0x7fffffffLL || N > 0x3fffffffLL || M % G != 0;
}

template <typename A>
int launch_rows(void (*kernel)(const A), int threads, size_t smem, int64_t ctas, const A& args,
                cudaStream_t s) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return TILEOPS_ELAUNCH;
  kernel<<<static_cast<unsigned>(ctas), threads, smem, s>>>(args);
  return launch_status();
}

}  // namespace
}  // namespace tileops
