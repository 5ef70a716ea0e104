// Sandwich norm: the norm after a block, the block's gate, the scaled residual
// and the norm before the next block, in one pass; and its backward pass.
//
// Per row of N (gate row g of the row's group):
//   p = norm(x) w1 + b1                      w1, b1: post_weight, post_bias
//   s = round_T(alpha residual + gate p)     -> residual_out
//   y = round_T(norm(s) w2 + b2)             w2, b2: pre_weight, pre_bias
// norm(v) = v rsqrt(mean v^2 + eps) (RMS) or (v - mean) rsqrt(var + eps)
// (LayerNorm, biased centred variance), statistics in fp32, those of the second
// norm over the ROUNDED s: the next block normalises what the stream holds,
// and the backward pass has only that (the rule of fused_add_layer_norm too).
//
// Backward, hats for normalised rows, ds the gradient of residual_out:
//   f   = dy w2;      ds' = ds + rstd_s (f - [mean f] - s^ mean(f s^))
//   e   = ds' gate w1; dx = rstd_x (e - [mean e] - x^ mean(e x^));  dres = alpha ds'
//   P_g = sum ds' x^, Q_g = sum ds' over the rows of group g
//   dw2 = sum dy s^, db2 = sum dy, dgate_g = w1 P_g + b1 Q_g,
//   dw1 = sum_g gate_g P_g, db1 = sum_g gate_g Q_g
// ([mean ..] terms: LayerNorm only).
//
// Both passes read each row once and write it once: persistent CTAs walk
// consecutive rows, a thread owns the same columns in every row (parameters and
// column sums stay in registers) and copies its own packets of the rows ahead into
// a private slot of a shared-memory ring.  A row costs one barrier, although it
// has two reductions one after another: the second of a row is exchanged together with the
// first of the next one.  A LayerNorm's mean and variance are taken warp by
// warp, centred there, and joined (Chan, Golub & LeVeque, "Updating formulae
// and a pairwise algorithm for computing sample variances", 1979).
//
// Measured (bf16, fp32 parameters): forward 8192 x 4096 52 us RMS, 54 us LayerNorm with
// biases and 8 gates (0.80 and 0.77 of the copy rate); backward 16384 x 4096 with its
// parameter sums 142 us (0.87), LayerNorm with biases 195 us (0.64).  Steps on the
// way: two barriers a row instead of one 60 and 193 us; scalar in place of packed
// arithmetic 72 and 234 us; the kind of norm tested at run time 55 and 149 us.
#include <algorithm>
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
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's packets of a row: packet j is the row's packet threadIdx.x + j kThreads, kV
// elements.  kAligned: rows of whole packets on 16-byte boundaries; otherwise
// packets are read and written element by element and the last one may be short.
template <typename T, int kThreads, int kPackets, bool kAligned>
struct Cols {
  static constexpr int kV = 16 / sizeof(T);
  static constexpr bool kWhole = kAligned;
  static __device__ __forceinline__ int first(int j) { return (threadIdx.x + j * kThreads) * kV; }
  // How many elements packet j has (all or none of an aligned row).
  static __device__ __forceinline__ int count(int j, int N) {
    const int left = N - first(j);
    return kAligned ? (left > 0 ? kV : 0) : max(0, min(kV, left));
  }
  static __device__ __forceinline__ void fetch(uint4* slot, const T* row, int j, int N) {
    if constexpr (kAligned) {
      if (first(j) < N) copy16(slot, row + first(j));
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
    if constexpr (kAligned) {
      st_stream(row + first(j), u);
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

// ---- forward ----
struct FwdArgs {
  const void *x, *res, *w1, *w2, *gate, *b1, *b2;
  void *y, *res_out;
  int64_t M;
  int N;
  int64_t rows_per_group;
  bool layer;
  float eps, alpha;
  bool vec;  // every parameter vector starts on a 16-byte boundary
};

template <typename T, typename W, int kThreads, int kPackets, int kStages, bool kAligned,
          bool kLayer>
__global__ void __launch_bounds__(kThreads) sn_fwd(const FwdArgs p) {
  using C = Cols<T, kThreads, kPackets, kAligned>;
  constexpr int kP = C::kP, kWarps = kThreads / 32;
  extern __shared__ uint4 ring[];  // [stage][x, residual][packet][thread]
  __shared__ WarpSums<4, kWarps> sums[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, N = p.N;
  constexpr bool layer = kLayer;
  const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.res);
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2),
          *gate = static_cast<const W*>(p.gate), *b1 = static_cast<const W*>(p.b1),
          *b2 = static_cast<const W*>(p.b2);
  const int64_t row0 = first_row(p.M, blockIdx.x, gridDim.x),
                end = first_row(p.M, blockIdx.x + 1, gridDim.x);
  auto slot = [&](int stage, int tensor, int j) {
    return ring + ((stage * 2 + tensor) * kPackets + j) * kThreads + threadIdx.x;
  };
  auto fetch = [&](int stage, int64_t row) {
    if (row < end)
#pragma unroll
      for (int j = 0; j < kPackets; ++j) {
        C::fetch(slot(stage, 0, j), x + row * N, j, N);
        C::fetch(slot(stage, 1, j), res + row * N, j, N);
      }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(s, row0 + s);

  int n[kPackets];
#pragma unroll
  for (int j = 0; j < kPackets; ++j) n[j] = C::count(j, N);
  float2 wg[kPackets][kP], bg[kPackets][kP], wn[kPackets][kP], bn[kPackets][kP];
  load_params<C>(wn, n, w2, 0.0f, p.vec);
  load_params<C>(bn, n, b2, 0.0f, p.vec);
  const float inv_n = 1.0f / static_cast<float>(N);
  const float mine = in_warp<C, kThreads, kPackets>(warp, N);
  const float inv_mine = mine > 0.0f ? 1.0f / mine : 0.0f;
  const int from = lane % kWarps;  // the warp whose sums this lane joins
  const float theirs = in_warp<C, kThreads, kPackets>(from, N);
  const float inv_theirs = theirs > 0.0f ? 1.0f / theirs : 0.0f;

  // x of the row in `stage`, zeros where the thread has no packet.
  auto read_x = [&](int stage, float2 (&v)[kPackets][kP]) {
#pragma unroll
    for (int j = 0; j < kPackets; ++j) {
      if (n[j] > 0)
        C::read(slot(stage, 0, j), v[j]);
      else
#pragma unroll
        for (int i = 0; i < kP; ++i) v[j][i] = both(0.0f);
    }
  };
  // One exchange: the moments of x of the next row and of s of this one -> their means and
  // 1 / deviations (mean_x, rstd_x, mean_s, rstd_s).
  int par = 0;
  auto exchange = [&](const float2(&xv)[kPackets][kP], const float2(&sv)[kPackets][kP]) {
    WarpSums<4, kWarps>& buf = sums[par];
    par ^= 1;
    float m[2] = {0.0f, 0.0f};
    if (layer) {
      m[0] = sum_of<C, kPackets>(xv);
      m[1] = sum_of<C, kPackets>(sv);
      warp_sums(m);
    }
    float q[2] = {squares_of<C, kPackets>(xv, n, layer, m[0] * inv_mine),
                  squares_of<C, kPackets>(sv, n, layer, m[1] * inv_mine)};
    warp_sums(q);
    if (lane == 0) {
      buf.v[0][warp] = m[0];
      buf.v[1][warp] = m[1];
      buf.v[2][warp] = q[0];
      buf.v[3][warp] = q[1];
    }
    __syncthreads();
    float mean[2] = {0.0f, 0.0f}, sq[2] = {buf.v[2][from], buf.v[3][from]};
    if (layer) {
      const float sum[2] = {buf.v[0][from], buf.v[1][from]};
      mean[0] = sum[0];
      mean[1] = sum[1];
      over_warps<kWarps>(mean);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mean[k] *= inv_n;
        const float d = sum[k] * inv_theirs - mean[k];
        sq[k] = fmaf(theirs * d, d, sq[k]);
      }
    }
    over_warps<kWarps>(sq);
    return make_float4(mean[0], rsqrtf(fmaf(sq[0], inv_n, p.eps)), mean[1],
                       rsqrtf(fmaf(sq[1], inv_n, p.eps)));
  };

  int stage = 0;
  int64_t next_group = row0;  // the row that starts another gate
  float2 v[kPackets][kP], xv[kPackets][kP];  // s of the row, x of the next one
  copies_wait<kStages - 2>();
  read_x(0, xv);
  float4 stat = exchange(xv, xv);
  for (int64_t row = row0; row < end; ++row) {
    if (row >= next_group) {
      const int64_t g = row / p.rows_per_group;
      next_group = (g + 1) * p.rows_per_group;
      float2 ga[kPackets][kP];
      load_params<C>(ga, n, gate ? gate + g * N : nullptr, 1.0f, p.vec);
      load_params<C>(wg, n, w1, 0.0f, p.vec);
      load_params<C>(bg, n, b1, 0.0f, p.vec);
      multiply<C>(wg, ga);
      multiply<C>(bg, ga);
    }
    T* out = static_cast<T*>(p.res_out) + row * N;
#pragma unroll
    for (int j = 0; j < kPackets; ++j) {
      if (n[j] > 0) {
        float2 r[kP];
        C::read(slot(stage, 1, j), r);
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          const float2 hat = normed<layer>(xv[j][i], stat.x, stat.y);
          v[j][i] = ffma2(both(p.alpha), r[i], ffma2(hat, wg[j][i], bg[j][i]));
          if (!kAligned && 2 * i >= n[j]) v[j][i].x = 0.0f;
          if (!kAligned && 2 * i + 1 >= n[j]) v[j][i].y = 0.0f;
        }
        C::write(out, j, N, v[j]);
        C::round(v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < kP; ++i) v[j][i] = both(0.0f);
      }
    }
    fetch(stage == 0 ? kStages - 1 : stage - 1, row + kStages - 1);
    copies_wait<kStages - 2>();
    stage = stage + 1 == kStages ? 0 : stage + 1;
    read_x(stage, xv);  // past the last row: what an earlier one left there, unused
    stat = exchange(xv, v);
    T* yr = static_cast<T*>(p.y) + row * N;
#pragma unroll
    for (int j = 0; j < kPackets; ++j) {
      if (n[j] > 0) {
#pragma unroll
        for (int i = 0; i < kP; ++i)
          v[j][i] = ffma2(normed<layer>(v[j][i], stat.z, stat.w), wn[j][i], bn[j][i]);
        C::write(yr, j, N, v[j]);
      }
    }
  }
  copies_wait<0>();
}

// ---- backward ----
struct BwdArgs {
  const void *dy, *ds, *x, *s, *w1, *w2, *gate;
  void *dx, *dres;
  float* part;
  int64_t M;
  int N;
  int64_t rows_per_group;
  bool layer;
  float eps, alpha;
  bool vec;  // every parameter vector starts on a 16-byte boundary
};

// Column sums of one stretch of rows (one CTA, one group): kBias ? P, Q, R, S : P, R, rows of N.
// Stretch (c, g) of CTA c and group g lies at index c + g, which grows from one
// stretch to the next, so no two share an index.
__device__ __forceinline__ float* stretch(float* part, int64_t c, int64_t g, int sums, int N) {
  return part + (c + g) * sums * N;
}

template <typename T, typename W, int kThreads, int kPackets, int kStages, int kCtas, bool kAligned,
          bool kBias, bool kLayer>
__global__ void __launch_bounds__(kThreads, kCtas) sn_bwd(const BwdArgs p) {
  using C = Cols<T, kThreads, kPackets, kAligned>;
  constexpr int kP = C::kP, kWarps = kThreads / 32, kSums = kBias ? 4 : 2;
  extern __shared__ uint4 ring[];  // [stage][x, s, dy, ds][packet][thread]
  __shared__ WarpSums<8, kWarps> sums[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, N = p.N;
  constexpr bool layer = kLayer;
  const T *x = static_cast<const T*>(p.x), *s = static_cast<const T*>(p.s),
          *dy = static_cast<const T*>(p.dy), *ds = static_cast<const T*>(p.ds);
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2),
          *gate = static_cast<const W*>(p.gate);
  const int64_t row0 = first_row(p.M, blockIdx.x, gridDim.x),
                end = first_row(p.M, blockIdx.x + 1, gridDim.x);
  auto slot = [&](int stage, int tensor, int j) {
    return ring + ((stage * 4 + tensor) * kPackets + j) * kThreads + threadIdx.x;
  };
  auto fetch = [&](int stage, int64_t row) {
    if (row < end)
#pragma unroll
      for (int j = 0; j < kPackets; ++j) {
        C::fetch(slot(stage, 0, j), x + row * N, j, N);
        C::fetch(slot(stage, 1, j), s + row * N, j, N);
        C::fetch(slot(stage, 2, j), dy + row * N, j, N);
        if (ds) C::fetch(slot(stage, 3, j), ds + row * N, j, N);
      }
    copies_commit();
  };
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) fetch(st, row0 + st);

  int n[kPackets];
#pragma unroll
  for (int j = 0; j < kPackets; ++j) n[j] = C::count(j, N);
  float2 wg[kPackets][kP], wn[kPackets][kP];
  float2 P[kPackets][kP], R[kPackets][kP], Q[kBias ? kPackets : 1][kP], S[kBias ? kPackets : 1][kP];
  load_params<C>(wn, n, w2, 0.0f, p.vec);
  auto clear = [&] {
#pragma unroll
    for (int j = 0; j < kPackets; ++j)
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        P[j][i] = R[j][i] = both(0.0f);
        if (kBias) Q[j][i] = S[j][i] = both(0.0f);
      }
  };
  clear();
  const float inv_n = 1.0f / static_cast<float>(N);
  const float mine = in_warp<C, kThreads, kPackets>(warp, N);
  const float inv_mine = mine > 0.0f ? 1.0f / mine : 0.0f;
  const int from = lane % kWarps;
  const float theirs = in_warp<C, kThreads, kPackets>(from, N);
  const float inv_theirs = theirs > 0.0f ? 1.0f / theirs : 0.0f;
  auto give = [&](int64_t g) {  // the column sums of the rows so far, which are of group g
    float* to = stretch(p.part, blockIdx.x, g, kSums, N);
    auto put = [&](int which, const float2& v, const float2& w, int c, int left) {
      float* at = to + which * static_cast<int64_t>(N) + c;
      if constexpr (kAligned) {
        if (left > 0) *reinterpret_cast<float4*>(at) = make_float4(v.x, v.y, w.x, w.y);
      } else {
        if (left > 0) at[0] = v.x;
        if (left > 1) at[1] = v.y;
        if (left > 2) at[2] = w.x;
        if (left > 3) at[3] = w.y;
      }
    };
#pragma unroll
    for (int j = 0; j < kPackets; ++j)
#pragma unroll
      for (int i = 0; i < kP; i += 2) {
        const int c = C::first(j) + 2 * i, left = n[j] - 2 * i;
        put(0, P[j][i], P[j][i + 1], c, left);
        put(1, R[j][i], R[j][i + 1], c, left);
        if constexpr (kBias) {
          put(2, Q[j][i], Q[j][i + 1], c, left);
          put(3, S[j][i], S[j][i + 1], c, left);
        }
      }
    clear();
  };

  // One exchange: of the row in `stage` the statistics of x and s, and of f = dy w2 with the
  // centred s; of the row before it E = sum e and Ex = sum e x^ (the thread's
  // sums), which come back over the CTA.
  struct Stats {
    float mean_x, rx, mean_s, rs, mean_f, mean_fs;
  };
  int par = 0;
  auto exchange = [&](int stage, float& E, float& Ex) {
    WarpSums<8, kWarps>& buf = sums[par];
    par ^= 1;
    // The row's packets are read from the ring in each pass: held in registers they would
    // cost a second resident CTA.
    float m[2] = {0.0f, 0.0f};
    if (layer) {
#pragma unroll
      for (int j = 0; j < kPackets; ++j)
        if (n[j] > 0) {
          float2 xv[1][kP], sv[1][kP];
          C::read(slot(stage, 0, j), xv[0]);
          C::read(slot(stage, 1, j), sv[0]);
          m[0] += sum_of<C, 1>(xv);
          m[1] += sum_of<C, 1>(sv);
        }
      warp_sums(m);
    }
    const float mean_xw = m[0] * inv_mine, mean_sw = m[1] * inv_mine;
    float2 F2 = both(0.0f), Fs2 = both(0.0f);
    float q[4] = {0.0f, 0.0f, 0.0f, Ex};
#pragma unroll
    for (int j = 0; j < kPackets; ++j)
      if (n[j] > 0) {
        float2 xv[1][kP], sv[1][kP], g[kP];
        const int one[1] = {n[j]};
        C::read(slot(stage, 0, j), xv[0]);
        C::read(slot(stage, 1, j), sv[0]);
        C::read(slot(stage, 2, j), g);
        q[0] += squares_of<C, 1>(xv, one, layer, mean_xw);
        q[1] += squares_of<C, 1>(sv, one, layer, mean_sw);
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          const float2 f = fmul2(g[i], wn[j][i]);
          if (layer) F2 = fadd2(F2, f);
          Fs2 = ffma2(f, layer ? fadd2(sv[0][i], both(-mean_sw)) : sv[0][i], Fs2);
        }
      }
    q[2] = total(Fs2);
    float l[2] = {total(F2), E};
    warp_sums(q);
    if (layer) warp_sums(l);
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) buf.v[k][warp] = q[k];
      buf.v[4][warp] = m[0];
      buf.v[5][warp] = m[1];
      buf.v[6][warp] = l[0];
      buf.v[7][warp] = l[1];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = buf.v[k][from];
    float mean[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of x, s, f; and E
    if (layer) {
      const float sum_x = buf.v[4][from], sum_s = buf.v[5][from], f = buf.v[6][from];
      mean[0] = sum_x;
      mean[1] = sum_s;
      mean[2] = f;
      mean[3] = buf.v[7][from];
      over_warps<kWarps>(mean);
      mean[0] *= inv_n;
      mean[1] *= inv_n;
      mean[2] *= inv_n;
      const float ex = sum_x * inv_theirs - mean[0], es = sum_s * inv_theirs - mean[1];
      q[0] = fmaf(theirs * ex, ex, q[0]);
      q[1] = fmaf(theirs * es, es, q[1]);
      q[2] = fmaf(f, es, q[2]);
    }
    over_warps<kWarps>(q);
    E = mean[3];
    Ex = q[3];
    Stats st;
    st.mean_x = mean[0];
    st.mean_s = mean[1];
    st.mean_f = mean[2];
    st.rx = rsqrtf(fmaf(q[0], inv_n, p.eps));
    st.rs = rsqrtf(fmaf(q[1], inv_n, p.eps));
    st.mean_fs = q[2] * inv_n * st.rs;
    return st;
  };

  int stage = 0;
  int64_t group = row0 / p.rows_per_group, next_group = row0;
  float E = 0.0f, Ex = 0.0f;
  copies_wait<kStages - 2>();
  Stats st = exchange(0, E, Ex);
  for (int64_t row = row0; row < end; ++row) {
    if (row >= next_group) {
      if (row > row0) give(group);
      group = row / p.rows_per_group;
      next_group = (group + 1) * p.rows_per_group;
      float2 ga[kPackets][kP];
      load_params<C>(ga, n, gate ? gate + group * N : nullptr, 1.0f, p.vec);
      load_params<C>(wg, n, w1, 0.0f, p.vec);
      multiply<C>(wg, ga);
    }
    // ds' and the sums for dx; e is kept for it.
    float2 ev[kPackets][kP];
    T* dres = static_cast<T*>(p.dres) + row * N;
    float2 E2 = both(0.0f), Ex2 = both(0.0f);
#pragma unroll
    for (int j = 0; j < kPackets; ++j) {
      if (n[j] > 0) {
        float2 t[kP], g[kP], xv[kP], sv[kP];
        C::read(slot(stage, 0, j), xv);
        C::read(slot(stage, 1, j), sv);
        C::read(slot(stage, 2, j), g);
        if (ds) {
          C::read(slot(stage, 3, j), t);
        } else {
#pragma unroll
          for (int i = 0; i < kP; ++i) t[i] = both(0.0f);
        }
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          const float2 hat = normed<layer>(sv[i], st.mean_s, st.rs);
          const float2 xh = normed<layer>(xv[i], st.mean_x, st.rx);
          const float2 off = layer ? ffma2(hat, both(-st.mean_fs), both(-st.mean_f))
                                   : fmul2(hat, both(-st.mean_fs));
          const float2 f = ffma2(g[i], wn[j][i], off);
          t[i] = ffma2(both(st.rs), f, t[i]);
          if (!kAligned && 2 * i >= n[j]) t[i].x = 0.0f;
          if (!kAligned && 2 * i + 1 >= n[j]) t[i].y = 0.0f;
          R[j][i] = ffma2(g[i], hat, R[j][i]);
          P[j][i] = ffma2(t[i], xh, P[j][i]);
          if (kBias) {
            Q[j][i] = fadd2(Q[j][i], t[i]);
            S[j][i] = fadd2(S[j][i], g[i]);
          }
          const float2 e = fmul2(t[i], wg[j][i]);
          if (layer) E2 = fadd2(E2, e);
          Ex2 = ffma2(e, xh, Ex2);
          t[i] = fmul2(both(p.alpha), t[i]);
          ev[j][i] = e;
        }
        C::write(dres, j, N, t);
      }
    }
    E = total(E2);
    Ex = total(Ex2);
    const float rx = st.rx, mean_x = st.mean_x;
    const int here = stage;
    fetch(stage == 0 ? kStages - 1 : stage - 1, row + kStages - 1);
    copies_wait<kStages - 2>();
    stage = stage + 1 == kStages ? 0 : stage + 1;
    st = exchange(stage, E, Ex);  // past the last row: of what an earlier one left there, unused
    // dx = rx (e - mean e - x^ mean(e x^)), x^ = (x - mean) rx
    const float mean_e = E * inv_n, slope = -Ex * inv_n * rx;
    T* dx = static_cast<T*>(p.dx) + row * N;
#pragma unroll
    for (int j = 0; j < kPackets; ++j) {
      if (n[j] > 0) {
        float2 o[kP];
        C::read(slot(here, 0, j), o);
#pragma unroll
        for (int i = 0; i < kP; ++i)
          o[i] = fmul2(both(rx), layer ? ffma2(fadd2(o[i], both(-mean_x)), both(slope),
                                               fadd2(ev[j][i], both(-mean_e)))
                                       : ffma2(o[i], both(slope), ev[j][i]));
        C::write(dx, j, N, o);
      }
    }
  }
  if (row0 < end) give(group);
  copies_wait<0>();
}

// Gradients of the parameters from the column sums of the stretches, added in a fixed
// order: 32 columns a CTA, kSlices threads a column.  With few groups the slices
// share the stretches of each group; with many, each takes whole groups.
constexpr int kSlices = 32;

template <typename W>
__global__ void __launch_bounds__(32 * kSlices)
    sn_params(const float* part, const W* w1, const W* gate, const W* b1, W* dw1, W* dw2, W* dgate,
              W* db1, W* db2, int64_t M, int N, int64_t G, int C, int sums) {
  __shared__ float red[4][kSlices][32], out[4][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const bool in = c < N;
  const float w1c = in ? Cvt<W>::to_f(w1[c]) : 0.0f, b1c = in ? param(b1, c, 0.0f) : 0.0f;
  const int64_t rpg = M / G;
  const bool by_group = G >= kSlices;
  // The CTA that has row r: the last one whose rows start at or before it.
  auto cta_of = [&](int64_t r) {
    int k = static_cast<int>(r * C / M);
    while (k + 1 < C && first_row(M, k + 1, C) <= r) ++k;
    while (first_row(M, k, C) > r) --k;
    return k;
  };
  auto across = [&](float (&v)[4]) {  // sums over the slices, in every thread
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < sums) red[q][slice][lane] = v[q];
    __syncthreads();
    if (slice < sums) {  // slice q adds up sum q
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kSlices; ++i) sum += red[slice][i][lane];
      out[slice][lane] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < sums) v[q] = out[q][lane];
  };
  float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // dw1, dw2, db1, db2
  for (int64_t g = by_group ? slice : 0; g < G; g += by_group ? kSlices : 1) {
    const int c0 = g == 0 ? 0 : cta_of(g * rpg), c1 = g == G - 1 ? C - 1 : cta_of((g + 1) * rpg - 1);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // P, R, Q, S
    if (in)
#pragma unroll 4
      for (int k = c0 + (by_group ? 0 : slice); k <= c1; k += by_group ? 1 : kSlices) {
        const float* p = part + (k + g) * sums * N + c;
        v[0] += p[0];
        v[1] += p[N];
        if (sums == 4) {
          v[2] += p[2 * static_cast<int64_t>(N)];
          v[3] += p[3 * static_cast<int64_t>(N)];
        }
      }
    if (!by_group) across(v);
    const float ga = in ? param(gate, g * N + c, 1.0f) : 0.0f;
    if (in && dgate && (by_group || slice == 0))
      dgate[g * N + c] = Cvt<W>::from_f(w1c * v[0] + b1c * v[2]);
    total[0] = fmaf(ga, v[0], total[0]);
    total[1] += v[1];
    total[2] = fmaf(ga, v[2], total[2]);
    total[3] += v[3];
  }
  if (by_group) across(total);
  if (in && slice == 0) {
    dw1[c] = Cvt<W>::from_f(total[0]);
    dw2[c] = Cvt<W>::from_f(total[1]);
    if (db1) db1[c] = Cvt<W>::from_f(total[2]);
    if (db2) db2[c] = Cvt<W>::from_f(total[3]);
  }
}

// ---- rows too wide for a thread's registers ----
// Passes over the row that read it again from L2.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  __syncthreads();  // `red` may still be read by the previous reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarps ? red[lane] : 0.0f);
}

// mean and rstd of a row read through `at`.
template <typename F>
__device__ __forceinline__ float2 row_stats(F at, int64_t N, bool layer, float eps, float* red) {
  float mean = 0.0f, sq = 0.0f;
  if (layer) {
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < N; c += blockDim.x) sum += at(c);
    mean = block_sum(sum, red) / static_cast<float>(N);
  }
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float d = at(c) - mean;
    sq = fmaf(d, d, sq);
  }
  return make_float2(mean, 1.0f / sqrtf(block_sum(sq, red) / static_cast<float>(N) + eps));
}

template <typename T, typename W>
__global__ void __launch_bounds__(1024) sn_fwd_wide(const FwdArgs p) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x, N = p.N, g = row / p.rows_per_group;
  const T *xr = static_cast<const T*>(p.x) + row * N, *rr = static_cast<const T*>(p.res) + row * N;
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2),
          *gate = static_cast<const W*>(p.gate), *b1 = static_cast<const W*>(p.b1),
          *b2 = static_cast<const W*>(p.b2);
  T *sr = static_cast<T*>(p.res_out) + row * N, *yr = static_cast<T*>(p.y) + row * N;
  const float2 sx =
      row_stats([&](int64_t c) { return Cvt<T>::to_f(xr[c]); }, N, p.layer, p.eps, red);
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float v = (Cvt<T>::to_f(xr[c]) - sx.x) * sx.y * Cvt<W>::to_f(w1[c]) + param(b1, c, 0.0f);
    sr[c] = Cvt<T>::from_f(fmaf(p.alpha, Cvt<T>::to_f(rr[c]), param(gate, g * N + c, 1.0f) * v));
  }
  const float2 ss =
      row_stats([&](int64_t c) { return Cvt<T>::to_f(sr[c]); }, N, p.layer, p.eps, red);
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x)
    yr[c] = Cvt<T>::from_f((Cvt<T>::to_f(sr[c]) - ss.x) * ss.y * Cvt<W>::to_f(w2[c]) +
                           param(b2, c, 0.0f));
}

// One CTA a stretch of rows: each row's statistics, its outputs, then its share of the
// column sums, which stay in the workspace (a thread adds to its own columns).
template <typename T, typename W, bool kBias>
__global__ void __launch_bounds__(1024) sn_bwd_wide(const BwdArgs p) {
  constexpr int kSums = kBias ? 4 : 2;
  __shared__ float red[32];
  const int64_t N = p.N;
  const T *x = static_cast<const T*>(p.x), *s = static_cast<const T*>(p.s),
          *dy = static_cast<const T*>(p.dy), *ds = static_cast<const T*>(p.ds);
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2),
          *gate = static_cast<const W*>(p.gate);
  const float inv_n = 1.0f / static_cast<float>(N);
  const int64_t row0 = first_row(p.M, blockIdx.x, gridDim.x),
                end = first_row(p.M, blockIdx.x + 1, gridDim.x);
  int64_t group = -1;
  for (int64_t row = row0; row < end; ++row) {
    const int64_t g = row / p.rows_per_group, o = row * N;
    float* to = stretch(p.part, blockIdx.x, g, kSums, p.N);
    if (g != group)
      for (int64_t c = threadIdx.x; c < N; c += blockDim.x)
        for (int q = 0; q < kSums; ++q) to[q * N + c] = 0.0f;
    group = g;
    const float2 sx =
        row_stats([&](int64_t c) { return Cvt<T>::to_f(x[o + c]); }, N, p.layer, p.eps, red);
    const float2 ss =
        row_stats([&](int64_t c) { return Cvt<T>::to_f(s[o + c]); }, N, p.layer, p.eps, red);
    float f0 = 0.0f, f1 = 0.0f;
    for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
      const float f = Cvt<T>::to_f(dy[o + c]) * Cvt<W>::to_f(w2[c]);
      f0 += f;
      f1 = fmaf(f, (Cvt<T>::to_f(s[o + c]) - ss.x) * ss.y, f1);
    }
    const float mf = p.layer ? block_sum(f0, red) * inv_n : 0.0f;
    const float mfs = block_sum(f1, red) * inv_n;
    float e0 = 0.0f, e1 = 0.0f;
    for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
      const float hat = (Cvt<T>::to_f(s[o + c]) - ss.x) * ss.y, dyv = Cvt<T>::to_f(dy[o + c]);
      const float xh = (Cvt<T>::to_f(x[o + c]) - sx.x) * sx.y;
      const float t = (ds ? Cvt<T>::to_f(ds[o + c]) : 0.0f) +
                      ss.y * (dyv * Cvt<W>::to_f(w2[c]) - mf - hat * mfs);
      to[c] = fmaf(t, xh, to[c]);
      to[N + c] = fmaf(dyv, hat, to[N + c]);
      if (kBias) {
        to[2 * N + c] += t;
        to[3 * N + c] += dyv;
      }
      const float e = t * param(gate, g * N + c, 1.0f) * Cvt<W>::to_f(w1[c]);
      e0 += e;
      e1 = fmaf(e, xh, e1);
    }
    const float me = p.layer ? block_sum(e0, red) * inv_n : 0.0f;
    const float mex = block_sum(e1, red) * inv_n;
    for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
      const float hat = (Cvt<T>::to_f(s[o + c]) - ss.x) * ss.y;
      const float t = (ds ? Cvt<T>::to_f(ds[o + c]) : 0.0f) +
                      ss.y * (Cvt<T>::to_f(dy[o + c]) * Cvt<W>::to_f(w2[c]) - mf - hat * mfs);
      const float e = t * param(gate, g * N + c, 1.0f) * Cvt<W>::to_f(w1[c]);
      static_cast<T*>(p.dres)[o + c] = Cvt<T>::from_f(p.alpha * t);
      static_cast<T*>(p.dx)[o + c] = Cvt<T>::from_f(
          sx.y * (e - me - (Cvt<T>::to_f(x[o + c]) - sx.x) * sx.y * mex));
    }
  }
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

bool bad_shape(int64_t M, int64_t N, int64_t G) {
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

// CTAs an SM of the backward pass: as many as their registers allow (each adds a stretch of
// column sums to write and read).  With biases there are twice the sums, and a row of
// 4096 takes more than the 128 registers a thread of two CTAs has (16384 x 4096
// bf16, before the norms were kernels of their own: two CTAs 152 us without and 284 us
// with biases, one 165 and 225 us).
int64_t ctas_per_sm(int64_t N, bool bias) {
  return N <= 1024 ? 4 : (N <= 2048 ? 2 : (N <= 4096 && !bias ? 2 : 1));
}
constexpr int kMaxSms = 256;  // workspace: more than any device of this architecture has

template <typename T, typename W, bool kAligned, bool kLayer>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  const int64_t packets = (a.N + 16 / sizeof(T) - 1) / (16 / sizeof(T));
  // per: CTAs an SM that fit; more rows ahead where a row is short.
  auto go = [&](auto kernel, int threads, int per_thread, int stages, int per) {
    return launch_rows(kernel, threads, static_cast<size_t>(stages) * 2 * per_thread * threads * 16,
                       std::min<int64_t>(a.M, static_cast<int64_t>(sm_count()) * per), a, s);
  };
  if (packets <= 64) return go(sn_fwd<T, W, 64, 1, 8, kAligned, kLayer>, 64, 1, 8, 12);
  if (packets <= 128) return go(sn_fwd<T, W, 128, 1, 6, kAligned, kLayer>, 128, 1, 6, 6);
  if (packets <= 256) return go(sn_fwd<T, W, 256, 1, 4, kAligned, kLayer>, 256, 1, 4, 3);
  if (packets <= 512) return go(sn_fwd<T, W, 256, 2, 4, kAligned, kLayer>, 256, 2, 4, 2);
  if (packets <= 1024) return go(sn_fwd<T, W, 512, 2, 3, kAligned, kLayer>, 512, 2, 3, 1);
  sn_fwd_wide<T, W><<<static_cast<unsigned>(a.M), 1024, 0, s>>>(a);
  return launch_status();
}

template <typename T, typename W, bool kAligned, bool kBias, bool kLayer>
int launch_bwd(const BwdArgs& a, int64_t ctas, cudaStream_t s) {
  const int64_t packets = (a.N + 16 / sizeof(T) - 1) / (16 / sizeof(T));
  auto go = [&](auto kernel, int threads, int per_thread, int stages) {
    return launch_rows(kernel, threads, static_cast<size_t>(stages) * 4 * per_thread * threads * 16,
                       ctas, a, s);
  };
  if (packets <= 128) return go(sn_bwd<T, W, 128, 1, 6, 4, kAligned, kBias, kLayer>, 128, 1, 6);
  if (packets <= 256) return go(sn_bwd<T, W, 256, 1, 5, 2, kAligned, kBias, kLayer>, 256, 1, 5);
  if (packets <= 512) {
    if constexpr (kBias)
      return go(sn_bwd<T, W, 256, 2, 4, 1, kAligned, kBias, kLayer>, 256, 2, 4);
    else
      return go(sn_bwd<T, W, 256, 2, 3, 2, kAligned, kBias, kLayer>, 256, 2, 3);
  }
  if (packets <= 1024) return go(sn_bwd<T, W, 512, 2, 3, 1, kAligned, kBias, kLayer>, 512, 2, 3);
  sn_bwd_wide<T, W, kBias><<<static_cast<unsigned>(ctas), 1024, 0, s>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace tileops

using namespace tileops;

extern "C" int tileops_sandwich_norm_fwd(const void* x, const void* residual,
                                         const void* post_weight, const void* pre_weight,
                                         const void* gate, const void* post_bias,
                                         const void* pre_bias, void* y, void* residual_out,
                                         int64_t M, int64_t N, int64_t gate_rows, int norm,
                                         double eps, double residual_scale, int dtype,
                                         int affine_dtype, void* stream) {
  if (bad_shape(M, N, gate_rows)) return TILEOPS_EBADSHAPE;
  if (norm != TILEOPS_NORM_RMS && norm != TILEOPS_NORM_LAYER) return TILEOPS_EINVAL;
  if (M == 0) return TILEOPS_OK;
  if (!x || !residual || !post_weight || !pre_weight || !y || !residual_out)
    return TILEOPS_EINVAL;
  const FwdArgs args{x, residual, post_weight, pre_weight, gate, post_bias, pre_bias, y,
                     residual_out, M, static_cast<int>(N), M / gate_rows,
                     norm == TILEOPS_NORM_LAYER, static_cast<float>(eps),
                     static_cast<float>(residual_scale),
                     aligned16(post_weight) && aligned16(pre_weight) && aligned16(gate) &&
                         aligned16(post_bias) && aligned16(pre_bias)};
  return with_types(dtype, affine_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const bool aligned = N * sizeof(T) % 16 == 0 && aligned16(x) && aligned16(residual) &&
                         aligned16(y) && aligned16(residual_out);
    auto go = [&](auto whole, auto layer) {
      return launch_fwd<T, W, whole.value, layer.value>(args, as_stream(stream));
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (args.layer) return aligned ? go(Yes(), Yes()) : go(No(), Yes());
    return aligned ? go(Yes(), No()) : go(No(), No());
  });
}

extern "C" int64_t tileops_sandwich_norm_bwd_workspace_bytes(int64_t M, int64_t N,
                                                             int64_t gate_rows, int has_bias) {
  if (bad_shape(M, N, gate_rows)) return -1;
  return (std::min<int64_t>(M, kMaxSms * ctas_per_sm(N, has_bias)) + gate_rows) * (has_bias ? 4 : 2) * N * 4;
}

extern "C" int tileops_sandwich_norm_bwd(const void* dy, const void* d_residual_out, const void* x,
                                         const void* residual_out, const void* post_weight,
                                         const void* pre_weight, const void* gate,
                                         const void* post_bias, void* dx, void* d_residual,
                                         void* d_post_weight, void* d_pre_weight, void* d_gate,
                                         void* d_post_bias, void* d_pre_bias, void* workspace,
                                         int64_t M, int64_t N, int64_t gate_rows, int norm,
                                         double eps, double residual_scale, int dtype,
                                         int affine_dtype, void* stream) {
  if (bad_shape(M, N, gate_rows)) return TILEOPS_EBADSHAPE;
  if (norm != TILEOPS_NORM_RMS && norm != TILEOPS_NORM_LAYER) return TILEOPS_EINVAL;
  if (M == 0) return TILEOPS_EBADSHAPE;
  if (!dy || !x || !residual_out || !post_weight || !pre_weight || !dx || !d_residual ||
      !d_post_weight || !d_pre_weight || !workspace || (d_gate && !gate) ||
      (d_post_bias && !post_bias))
    return TILEOPS_EINVAL;
  cudaStream_t st = as_stream(stream);
  // The gate's gradient takes Q when there is a post_bias, whether or not that has one.
  const bool bias = post_bias || d_pre_bias;
  float* part = static_cast<float*>(workspace);
  const BwdArgs args{dy, d_residual_out, x, residual_out, post_weight, pre_weight, gate, dx,
                     d_residual, part, M, static_cast<int>(N), M / gate_rows,
                     norm == TILEOPS_NORM_LAYER, static_cast<float>(eps),
                     static_cast<float>(residual_scale),
                     aligned16(post_weight) && aligned16(pre_weight) && aligned16(gate)};
  const int64_t ctas = std::min<int64_t>(M, std::min(sm_count(), kMaxSms) * ctas_per_sm(N, bias));
  return with_types(dtype, affine_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const bool aligned = N * sizeof(T) % 16 == 0 && aligned16(dy) && aligned16(d_residual_out) &&
                         aligned16(x) && aligned16(residual_out) && aligned16(dx) &&
                         aligned16(d_residual);
    using Yes = std::true_type;
    using No = std::false_type;
    auto go = [&](auto whole, auto biased) {
      return args.layer ? launch_bwd<T, W, whole.value, biased.value, true>(args, ctas, st)
                        : launch_bwd<T, W, whole.value, biased.value, false>(args, ctas, st);
    };
    const int status = aligned ? (bias ? go(Yes(), Yes()) : go(Yes(), No()))
                               : (bias ? go(No(), Yes()) : go(No(), No()));
    if (status != TILEOPS_OK) return status;
    auto par = [](const void* p) { return static_cast<const W*>(p); };
    auto out = [](void* p) { return static_cast<W*>(p); };
    sn_params<W><<<static_cast<unsigned>((N + 31) / 32), 32 * kSlices, 0, st>>>(
        part, par(post_weight), par(gate), par(post_bias), out(d_post_weight), out(d_pre_weight),
        out(d_gate), out(d_post_bias), out(d_pre_bias), M, static_cast<int>(N), gate_rows,
        static_cast<int>(ctas), bias ? 4 : 2);
    return launch_status();
  });
}
