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
#include "common.cuh"

namespace tileops {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA; every thread gets the total.  `red` holds 32 floats.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  __syncthreads();  // `red` may still be read by the previous reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarps ? red[lane] : 0.0f);
}

template <typename W>
__device__ __forceinline__ float param(const W* p, int64_t i, float otherwise) {
  return p ? Cvt<W>::to_f(p[i]) : otherwise;
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
__global__ void __launch_bounds__(256)
    sn_fwd_simple(const T* x, const T* res, const W* w1, const W* w2, const W* gate, const W* b1,
                  const W* b2, T* y, T* res_out, int64_t N, int64_t rows_per_group, bool layer,
                  float eps, float alpha) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x, g = row / rows_per_group;
  const T* xr = x + row * N;
  T* sr = res_out + row * N;
  const float2 sx =
      row_stats([&](int64_t c) { return Cvt<T>::to_f(xr[c]); }, N, layer, eps, red);
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float p = (Cvt<T>::to_f(xr[c]) - sx.x) * sx.y * Cvt<W>::to_f(w1[c]) + param(b1, c, 0.0f);
    sr[c] = Cvt<T>::from_f(fmaf(alpha, Cvt<T>::to_f(res[row * N + c]),
                                param(gate, g * N + c, 1.0f) * p));
  }
  const float2 ss =
      row_stats([&](int64_t c) { return Cvt<T>::to_f(sr[c]); }, N, layer, eps, red);
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x)
    y[row * N + c] = Cvt<T>::from_f((Cvt<T>::to_f(sr[c]) - ss.x) * ss.y * Cvt<W>::to_f(w2[c]) +
                                    param(b2, c, 0.0f));
}

struct RowStats {
  float mean_x, rstd_x, mean_s, rstd_s, mean_f, mean_fs;
};

template <typename T, typename W>
__global__ void __launch_bounds__(256)
    sn_bwd_rows_simple(const T* dy, const T* ds, const T* x, const T* s, const W* w1, const W* w2,
                       const W* gate, T* dx, T* dres, RowStats* stats, int64_t N,
                       int64_t rows_per_group, bool layer, float eps, float alpha) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x, g = row / rows_per_group, o = row * N;
  const float inv_n = 1.0f / static_cast<float>(N);
  const float2 sx = row_stats([&](int64_t c) { return Cvt<T>::to_f(x[o + c]); }, N, layer, eps, red);
  const float2 ss = row_stats([&](int64_t c) { return Cvt<T>::to_f(s[o + c]); }, N, layer, eps, red);
  float f0 = 0.0f, f1 = 0.0f;
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float f = Cvt<T>::to_f(dy[o + c]) * Cvt<W>::to_f(w2[c]);
    f0 += f;
    f1 += f * (Cvt<T>::to_f(s[o + c]) - ss.x) * ss.y;
  }
  const float mf = layer ? block_sum(f0, red) * inv_n : 0.0f, mfs = block_sum(f1, red) * inv_n;
  auto total = [&](int64_t c) {
    const float hat = (Cvt<T>::to_f(s[o + c]) - ss.x) * ss.y;
    const float f = Cvt<T>::to_f(dy[o + c]) * Cvt<W>::to_f(w2[c]);
    return (ds ? Cvt<T>::to_f(ds[o + c]) : 0.0f) + ss.y * (f - mf - hat * mfs);
  };
  float e0 = 0.0f, e1 = 0.0f;
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float e = total(c) * param(gate, g * N + c, 1.0f) * Cvt<W>::to_f(w1[c]);
    e0 += e;
    e1 += e * (Cvt<T>::to_f(x[o + c]) - sx.x) * sx.y;
  }
  const float me = layer ? block_sum(e0, red) * inv_n : 0.0f, mex = block_sum(e1, red) * inv_n;
  for (int64_t c = threadIdx.x; c < N; c += blockDim.x) {
    const float t = total(c), e = t * param(gate, g * N + c, 1.0f) * Cvt<W>::to_f(w1[c]);
    dres[o + c] = Cvt<T>::from_f(alpha * t);
    dx[o + c] = Cvt<T>::from_f(sx.y * (e - me - (Cvt<T>::to_f(x[o + c]) - sx.x) * sx.y * mex));
  }
  if (threadIdx.x == 0) stats[row] = RowStats{sx.x, sx.y, ss.x, ss.y, mf, mfs};
}

template <typename T, typename W>
__global__ void __launch_bounds__(128)
    sn_bwd_cols_simple(const T* dy, const T* ds, const T* x, const T* s, const W* w1, const W* w2,
                       const W* gate, const W* b1, const RowStats* stats, W* dw1, W* dw2, W* dgate,
                       W* db1, W* db2, int64_t M, int64_t N, int64_t G) {
  const int64_t c = blockIdx.x * 128ll + threadIdx.x;
  if (c >= N) return;
  const float w1c = Cvt<W>::to_f(w1[c]), w2c = Cvt<W>::to_f(w2[c]), b1c = param(b1, c, 0.0f);
  float aw1 = 0.0f, ab1 = 0.0f, R = 0.0f, S = 0.0f;
  for (int64_t g = 0; g < G; ++g) {
    float P = 0.0f, Q = 0.0f;
    for (int64_t row = g * (M / G); row < (g + 1) * (M / G); ++row) {
      const RowStats st = stats[row];
      const float dyv = Cvt<T>::to_f(dy[row * N + c]);
      const float hat = (Cvt<T>::to_f(s[row * N + c]) - st.mean_s) * st.rstd_s;
      const float t = (ds ? Cvt<T>::to_f(ds[row * N + c]) : 0.0f) +
                      st.rstd_s * (dyv * w2c - st.mean_f - hat * st.mean_fs);
      P = fmaf(t, (Cvt<T>::to_f(x[row * N + c]) - st.mean_x) * st.rstd_x, P);
      Q += t;
      R = fmaf(dyv, hat, R);
      S += dyv;
    }
    const float gc = param(gate, g * N + c, 1.0f);
    if (dgate) dgate[g * N + c] = Cvt<W>::from_f(w1c * P + b1c * Q);
    aw1 = fmaf(gc, P, aw1);
    ab1 = fmaf(gc, Q, ab1);
  }
  dw1[c] = Cvt<W>::from_f(aw1);
  dw2[c] = Cvt<W>::from_f(R);
  if (db1) db1[c] = Cvt<W>::from_f(ab1);
  if (db2) db2[c] = Cvt<W>::from_f(S);
}

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
  return M < 0 || N <= 0 || G < 1 || M > 0x7fffffffLL || N > 0x7fffffffLL || M % G != 0;
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
  return with_types(dtype, affine_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    sn_fwd_simple<T, W><<<static_cast<unsigned>(M), 256, 0, as_stream(stream)>>>(
        static_cast<const T*>(x), static_cast<const T*>(residual),
        static_cast<const W*>(post_weight), static_cast<const W*>(pre_weight),
        static_cast<const W*>(gate), static_cast<const W*>(post_bias),
        static_cast<const W*>(pre_bias), static_cast<T*>(y), static_cast<T*>(residual_out), N,
        M / gate_rows, norm == TILEOPS_NORM_LAYER, static_cast<float>(eps),
        static_cast<float>(residual_scale));
    return launch_status();
  });
}

extern "C" int64_t tileops_sandwich_norm_bwd_workspace_bytes(int64_t M, int64_t N,
                                                             int64_t gate_rows, int has_bias) {
  (void)has_bias;
  if (bad_shape(M, N, gate_rows)) return -1;
  return M * static_cast<int64_t>(sizeof(RowStats));
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
  return with_types(dtype, affine_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    RowStats* stats = static_cast<RowStats*>(workspace);
    auto in = [](const void* p) { return static_cast<const T*>(p); };
    auto par = [](const void* p) { return static_cast<const W*>(p); };
    auto out = [](void* p) { return static_cast<W*>(p); };
    sn_bwd_rows_simple<T, W><<<static_cast<unsigned>(M), 256, 0, st>>>(
        in(dy), in(d_residual_out), in(x), in(residual_out), par(post_weight), par(pre_weight),
        par(gate), static_cast<T*>(dx), static_cast<T*>(d_residual), stats, N, M / gate_rows,
        norm == TILEOPS_NORM_LAYER, static_cast<float>(eps), static_cast<float>(residual_scale));
    sn_bwd_cols_simple<T, W><<<static_cast<unsigned>((N + 127) / 128), 128, 0, st>>>(
        in(dy), in(d_residual_out), in(x), in(residual_out), par(post_weight), par(pre_weight),
        par(gate), par(post_bias), stats, out(d_post_weight), out(d_pre_weight), out(d_gate),
        out(d_post_bias), out(d_pre_bias), M, N, gate_rows);
    return launch_status();
  });
}
