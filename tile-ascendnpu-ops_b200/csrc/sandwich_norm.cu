// Sandwich norm: the norm after a block, the block's gate, the scaled residual
// and the norm before the next block, in one pass.  (Backward: sandwich_norm_bwd.cu.)
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
// column sums stay with it, in registers but for the spills named below) and copies its own
// packets of the rows ahead into a private slot of a shared-memory ring.  A row costs one
// barrier, although it has two reductions one after another: the second of a row is exchanged together with the
// first of the next one.  A LayerNorm's mean and variance are taken warp by
// warp, centred there, and joined (Chan, Golub & LeVeque, "Updating formulae
// and a pairwise algorithm for computing sample variances", 1979).
//
// Measured (bf16, fp32 parameters): forward 8192 x 4096 52 us RMS, 53 us LayerNorm with
// biases and 8 gates (0.80 and 0.78 of the copy rate); backward 16384 x 4096 with its
// parameter sums 143 us (0.87), LayerNorm with biases 195 us (0.64).  All fp32: 8192 x
// 4096 92 us (0.90) and 147 us (0.84).  Rows of 4097 to 8192 in 16 bits take 512 threads
// of 128 registers; backward with biases these spill 96 to 364 bytes a thread, up to 428 where
// copies are of 4 bytes (4096 x 8192 LayerNorm with biases 162 us, 0.38).  Steps on the
// way: two barriers a row instead of one 60 and 193 us; scalar in place of packed
// arithmetic 72 and 234 us; the kind of norm tested at run time 55 and 149 us.
#include "sandwich_norm.cuh"

namespace tileops {
namespace {

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

template <typename T, typename W, int kThreads, int kPackets, int kStages, int kBytes,
          bool kLayer>
__global__ void __launch_bounds__(kThreads) sn_fwd(const FwdArgs p) {
  using C = Cols<T, kThreads, kPackets, kBytes>;
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
          if (!C::kWhole && 2 * i >= n[j]) v[j][i].x = 0.0f;
          if (!C::kWhole && 2 * i + 1 >= n[j]) v[j][i].y = 0.0f;
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

template <typename T, typename W, int kV>
__global__ void __launch_bounds__(1024) sn_fwd_wide(const FwdArgs p) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x, N = p.N, g = row / p.rows_per_group;
  const int64_t first = static_cast<int64_t>(threadIdx.x) * kV, step = blockDim.x * kV;
  const T *xr = static_cast<const T*>(p.x) + row * N, *rr = static_cast<const T*>(p.res) + row * N;
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2),
          *gate = static_cast<const W*>(p.gate), *b1 = static_cast<const W*>(p.b1),
          *b2 = static_cast<const W*>(p.b2);
  T *sr = static_cast<T*>(p.res_out) + row * N, *yr = static_cast<T*>(p.y) + row * N;
  const float2 sx = row_stats<kV>(xr, N, p.layer, p.eps, red);
  float v[kV], r[kV], w[kV], o[kV], ga[kV];
  for (int64_t c = first; c < N; c += step) {
    load_cols<kV>(xr + c, v);
    load_cols<kV>(rr + c, r);
    load_vector<kV>(w1, c, 1.0f, p.vec, w);
    load_vector<kV>(b1, c, 0.0f, p.vec, o);
    load_vector<kV>(gate ? gate + g * N : nullptr, c, 1.0f, p.vec, ga);
#pragma unroll
    for (int i = 0; i < kV; ++i)
      v[i] = fmaf(p.alpha, r[i], ga[i] * fmaf((v[i] - sx.x) * sx.y, w[i], o[i]));
    store_cols<kV>(sr + c, v);
  }
  // (a thread reads back only what it wrote)
  const float2 ss = row_stats<kV>(sr, N, p.layer, p.eps, red);
  for (int64_t c = first; c < N; c += step) {
    load_cols<kV>(sr + c, v);
    load_vector<kV>(w2, c, 1.0f, p.vec, w);
    load_vector<kV>(b2, c, 0.0f, p.vec, o);
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = fmaf((v[i] - ss.x) * ss.y, w[i], o[i]);
    store_cols<kV>(yr + c, v);
  }
}

template <typename T, typename W, int kBytes, bool kLayer>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  const int64_t packets = (a.N + 16 / sizeof(T) - 1) / (16 / sizeof(T));
  // per: CTAs an SM that fit; more rows ahead where a row is short.
  auto go = [&](auto kernel, int threads, int per_thread, int stages, int per) {
    return launch_rows(kernel, threads, static_cast<size_t>(stages) * 2 * per_thread * threads * 16,
                       std::min<int64_t>(a.M, static_cast<int64_t>(sm_count()) * per), a, s);
  };
  if (packets <= 64) return go(sn_fwd<T, W, 64, 1, 8, kBytes, kLayer>, 64, 1, 8, 12);
  if (packets <= 128) return go(sn_fwd<T, W, 128, 1, 6, kBytes, kLayer>, 128, 1, 6, 6);
  if (packets <= 256) return go(sn_fwd<T, W, 256, 1, 4, kBytes, kLayer>, 256, 1, 4, 3);
  if (packets <= 512) return go(sn_fwd<T, W, 256, 2, 4, kBytes, kLayer>, 256, 2, 4, 2);
  if (packets <= 1024) return go(sn_fwd<T, W, 512, 2, 3, kBytes, kLayer>, 512, 2, 3, 1);
  sn_fwd_wide<T, W, kBytes == 16 ? 16 / sizeof(T) : 1><<<static_cast<unsigned>(a.M), 1024, 0, s>>>(a);
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
    return with_bytes<T>(N, {x, residual, y, residual_out}, [&](auto bytes) {
      return args.layer ? launch_fwd<T, W, bytes.value, true>(args, as_stream(stream))
                        : launch_fwd<T, W, bytes.value, false>(args, as_stream(stream));
    });
  });
}

