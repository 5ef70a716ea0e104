// Gated linear recurrence over channels: forward, backward and one decode step.
//
// Per channel d and token t, with input x, input gate i and decay gate r
// (logits) and a learned lambda per channel:
//   k     = c softplus(lambda)              >= 0
//   log a = -k sigmoid(r),  a = exp(log a),  m = sqrt(1 - a^2)
//   h_t   = a_t h_{t-1} + m_t sigmoid(i_t) x_t,   y_t = h_t     (h in fp32)
// Backward, G_t = dL/dh_t:
//   G_t   = dy_t + a_{t+1} G_{t+1}          (+ the final state's gradient)
//   dx    = G m sigma_i                     di = G m x sigma_i (1 - sigma_i)
//   dloga = a G h_{t-1} - G sigma_i x a^2 / m
//   dr    = -k sigma_r (1 - sigma_r) dloga  dlambda = -c sigmoid(lambda) sum sigma_r dloga
// Where m = 0 (a gate closed to the last bit) the second term of dloga is 0,
// its limit: it enters dr and dlambda as k sigma_r / m -> sqrt(k sigma_r / 2).
//
// Packed sequences (cu_seqlens): the first token of a sequence takes its
// predecessor from initial_state by selection, not by a zero factor, so
// infinities and NaN of one sequence never reach another.
#include <algorithm>

#include "common.cuh"
#include "device_error.cuh"

namespace tileops {
namespace {

constexpr int kSegment = TILEOPS_GLR_SEGMENT;  // tokens between saved states
constexpr float kLog2e = 1.4426950408889634f;

// ---- the gates of one element ----
struct Gates {
  float si, sr;  // sigmoid of the input gate and of the decay gate
  float a, m2;   // decay and 1 - a^2
};

__device__ __forceinline__ float sigmoid_f(float z) {
  return rcp_approx_f(1.0f + ex2_approx_f(-kLog2e * z));
}

// a and 1 - a^2 from log a <= 0.  Near zero both come from q = a - 1 = expm1(log a)
// (Taylor series to the sixth power: off by less than log_a^6 / 5040 = 5e-8 of q at
// -1/4): 1 - a^2 = -q (2 + q) has no cancellation, and 1 + q rounds once, where an
// approximate exponential's error would be carried along the whole sequence.
__device__ __forceinline__ void decay_from_log(float la, float& a, float& m2) {
  float p = fmaf(la, 1.0f / 720.0f, 1.0f / 120.0f);
  p = fmaf(la, p, 1.0f / 24.0f);
  p = fmaf(la, p, 1.0f / 6.0f);
  p = fmaf(la, p, 0.5f);
  p = fmaf(la, p, 1.0f);
  const float q = la * p;
  const float e = ex2_approx_f(kLog2e * la);
  const bool near = la > -0.25f;
  a = near ? 1.0f + q : e;
  m2 = near ? -q * (2.0f + q) : fmaf(-e, e, 1.0f);
}

__device__ __forceinline__ Gates gates_of(float i, float r, float k) {
  Gates g;
  g.si = sigmoid_f(i);
  g.sr = sigmoid_f(r);
  decay_from_log(-k * g.sr, g.a, g.m2);
  return g;
}

__device__ __forceinline__ float softplus_f(float z) {
  return fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z)));
}
// c softplus(lambda), with a NaN kept (fmaxf would drop it).
__device__ __forceinline__ float decay_rate(float lambda, float c) {
  return lambda != lambda ? lambda : c * softplus_f(lambda);
}

// ---- packed sequences ----
// The sequence token t belongs to: the last n with cu[n] <= t, in [0, N).
__device__ __forceinline__ int seq_of(const int32_t* cu, int N, int64_t t) {
  int lo = 0, hi = N;  // cu[lo] <= t (or lo = 0), cu[hi] > t (or hi = N)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

struct Strides {
  int64_t xb, xt, ib, it, rb, rt, gb, gt;  // x, input gate, decay gate, dy: batch and token
};

template <typename T>
__global__ void __launch_bounds__(128)
    glr_fwd_simple(const T* x, const T* ig, const T* rg, const float* lam, const float* h0,
                   const int32_t* cu, int N, T* y, float* hT, float* states, int64_t T_, int64_t D,
                   Strides st, float c) {
  const int64_t d = blockIdx.x * 128ll + threadIdx.x, b = blockIdx.y;
  if (d >= D) return;
  const float k = decay_rate(lam[d], c);
  const int64_t nseg = (T_ + kSegment - 1) / kSegment;
  if (cu)
    for (int n = 0; n < N; ++n)
      if (cu[n + 1] <= cu[n]) hT[n * D + d] = h0 ? h0[n * D + d] : 0.0f;
  float h = cu ? 0.0f : (h0 ? h0[b * D + d] : 0.0f);
  for (int64_t t = 0; t < T_; ++t) {
    if (states && t % kSegment == 0) states[(b * nseg + t / kSegment) * D + d] = h;
    int n = 0;
    if (cu) {
      n = seq_of(cu, N, t);
      if (cu[n] == t) h = h0 ? h0[n * D + d] : 0.0f;
    }
    const Gates g = gates_of(Cvt<T>::to_f(ig[b * st.ib + t * st.it + d]),
                             Cvt<T>::to_f(rg[b * st.rb + t * st.rt + d]), k);
    const float xv = Cvt<T>::to_f(x[b * st.xb + t * st.xt + d]);
    h = fmaf(g.a, h, sqrtf(g.m2) * g.si * xv);
    y[(b * T_ + t) * D + d] = Cvt<T>::from_f(h);
    if (cu && cu[n + 1] == t + 1) hT[n * D + d] = h;
  }
  if (!cu) hT[b * D + d] = h;
}

template <typename T>
__global__ void __launch_bounds__(128)
    glr_bwd_simple(const T* dy, const T* x, const T* ig, const T* rg, const float* lam,
                   const float* states, const float* h0, const float* dhT, const int32_t* cu, int N,
                   T* dx, T* di, T* dr, float* part, float* dh0, int64_t T_, int64_t D, Strides st,
                   float c) {
  const int64_t d = blockIdx.x * 128ll + threadIdx.x, b = blockIdx.y;
  if (d >= D) return;
  const float k = decay_rate(lam[d], c);
  const int64_t nseg = (T_ + kSegment - 1) / kSegment;
  if (cu)
    for (int n = 0; n < N; ++n)
      if (cu[n + 1] <= cu[n]) dh0[n * D + d] = dhT ? dhT[n * D + d] : 0.0f;
  float back = cu ? 0.0f : (dhT ? dhT[b * D + d] : 0.0f), dk = 0.0f;
  for (int64_t seg = nseg - 1; seg >= 0; --seg) {
    float hp[kSegment];
    float h = states[(b * nseg + seg) * D + d];
    const int64_t t0 = seg * kSegment;
    const int len = static_cast<int>(T_ - t0 < kSegment ? T_ - t0 : kSegment);
    for (int j = 0; j < len; ++j) {
      const int64_t t = t0 + j;
      if (cu) {
        const int n = seq_of(cu, N, t);
        if (cu[n] == t) h = h0 ? h0[n * D + d] : 0.0f;
      }
      hp[j] = h;
      const Gates g = gates_of(Cvt<T>::to_f(ig[b * st.ib + t * st.it + d]),
                               Cvt<T>::to_f(rg[b * st.rb + t * st.rt + d]), k);
      h = fmaf(g.a, h, sqrtf(g.m2) * g.si * Cvt<T>::to_f(x[b * st.xb + t * st.xt + d]));
    }
    for (int j = len - 1; j >= 0; --j) {
      const int64_t t = t0 + j;
      int n = 0;
      if (cu) {
        n = seq_of(cu, N, t);
        if (cu[n + 1] == t + 1) back = dhT ? dhT[n * D + d] : 0.0f;
      }
      const Gates g = gates_of(Cvt<T>::to_f(ig[b * st.ib + t * st.it + d]),
                               Cvt<T>::to_f(rg[b * st.rb + t * st.rt + d]), k);
      const float xv = Cvt<T>::to_f(x[b * st.xb + t * st.xt + d]);
      const float G = Cvt<T>::to_f(dy[b * st.gb + t * st.gt + d]) + back;
      const float m = sqrtf(g.m2), over_m = g.m2 > 0.0f ? 1.0f / m : 0.0f * g.m2;
      const float gx = G * m * g.si;
      const float dla = g.a * G * (hp[j] - g.a * g.si * xv * over_m);
      const int64_t o = (b * T_ + t) * D + d;
      dx[o] = Cvt<T>::from_f(gx);
      di[o] = Cvt<T>::from_f(gx * xv * (1.0f - g.si));
      dr[o] = Cvt<T>::from_f(-k * g.sr * (1.0f - g.sr) * dla);
      dk = fmaf(-g.sr, dla, dk);
      back = g.a * G;
      if (cu && cu[n] == t) dh0[n * D + d] = back;
    }
  }
  if (!cu) dh0[b * D + d] = back;
  part[b * D + d] = dk;
}

// dlambda = c sigmoid(lambda) sum of the partial sums, added in a fixed order.
__global__ void __launch_bounds__(128)
    glr_dparam(const float* part, const float* lam, float* dlam, int64_t parts, int64_t D, float c) {
  const int64_t d = blockIdx.x * 128ll + threadIdx.x;
  if (d >= D) return;
  float s = 0.0f;
  for (int64_t p = 0; p < parts; ++p) s += part[p * D + d];
  dlam[d] = s * c / (1.0f + expf(-lam[d]));
}

// cu_seqlens must be 0 = cu[0] <= ... <= cu[N] = total; reported otherwise.
__global__ void glr_check_seqlens(const int32_t* cu, int N, int64_t total, int* err) {
  bool bad = false;
  for (int n = threadIdx.x; n < N; n += blockDim.x) bad |= cu[n + 1] < cu[n];
  if (threadIdx.x == 0) bad |= cu[0] != 0 || cu[N] != total;
  if (bad) report_device_error(err, kErrBadSeqlens);
}

template <typename T>
__global__ void __launch_bounds__(128)
    glr_decode(const T* x, const T* ig, const T* rg, const float* lam, const float* h0, T* y,
               float* hn, int64_t D, Strides st, float c) {
  const int64_t d = blockIdx.x * 128ll + threadIdx.x, b = blockIdx.y;
  if (d >= D) return;
  const Gates g = gates_of(Cvt<T>::to_f(ig[b * st.ib + d]), Cvt<T>::to_f(rg[b * st.rb + d]),
                           decay_rate(lam[d], c));
  const float h = fmaf(g.a, h0[b * D + d], sqrtf(g.m2) * g.si * Cvt<T>::to_f(x[b * st.xb + d]));
  y[b * D + d] = Cvt<T>::from_f(h);
  hn[b * D + d] = h;
}

int64_t bwd_parts(int64_t batch, int64_t, int64_t) { return batch; }

// Sizes every kernel here indexes with: batch in a grid's y, 64-bit element offsets.
bool bad_shape(int64_t batch, int64_t seq_len, int64_t dim) {
  return batch < 0 || seq_len < 0 || dim < 0 || batch > 65535 || seq_len > 0x7fffffffLL ||
         dim > 0x7fffffffLL;
}

}  // namespace
}  // namespace tileops

using namespace tileops;

extern "C" int tileops_glr_fwd(const void* x, const void* input_gate, const void* decay_gate,
                               const float* decay_param, const float* initial_state,
                               const int32_t* cu_seqlens, int64_t num_seqs, void* y,
                               float* final_state, float* states, int64_t batch, int64_t seq_len,
                               int64_t dim, int64_t x_stride_b, int64_t x_stride_t,
                               int64_t i_stride_b, int64_t i_stride_t, int64_t r_stride_b,
                               int64_t r_stride_t, double decay_scale, int dtype, void* stream) {
  if (bad_shape(batch, seq_len, dim)) return TILEOPS_EBADSHAPE;
  if (cu_seqlens && (batch != 1 || num_seqs < 1 || num_seqs > 0x7ffffffeLL))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || dim == 0) return TILEOPS_OK;
  if (seq_len == 0) return TILEOPS_EBADSHAPE;
  if (!x || !input_gate || !decay_gate || !decay_param || !y || !final_state)
    return TILEOPS_EINVAL;
  cudaStream_t s = as_stream(stream);
  const Strides st{x_stride_b, x_stride_t, i_stride_b, i_stride_t, r_stride_b, r_stride_t, 0, 0};
  const dim3 grid(static_cast<unsigned>((dim + 127) / 128), static_cast<unsigned>(batch));
  const int N = static_cast<int>(num_seqs);
  const float c = static_cast<float>(decay_scale);
  if (cu_seqlens) glr_check_seqlens<<<1, 128, 0, s>>>(cu_seqlens, N, seq_len, device_error_ptr());
  auto go = [&](auto zero) {
    using T = decltype(zero);
    glr_fwd_simple<T><<<grid, 128, 0, s>>>(
        static_cast<const T*>(x), static_cast<const T*>(input_gate),
        static_cast<const T*>(decay_gate), decay_param, initial_state, cu_seqlens, N,
        static_cast<T*>(y), final_state, states, seq_len, dim, st, c);
    return launch_status();
  };
  switch (dtype) {
    case TILEOPS_DT_F32: return go(float());
    case TILEOPS_DT_F16: return go(__half());
    default: return go(__nv_bfloat16());
  }
}

extern "C" int64_t tileops_glr_bwd_workspace_bytes(int64_t batch, int64_t seq_len, int64_t dim) {
  if (bad_shape(batch, seq_len, dim)) return -1;
  return bwd_parts(batch, seq_len, dim) * dim * 4;
}

extern "C" int tileops_glr_bwd(const void* dy, const void* x, const void* input_gate,
                               const void* decay_gate, const float* decay_param,
                               const float* states, const float* initial_state,
                               const float* d_final_state, const int32_t* cu_seqlens,
                               int64_t num_seqs, void* dx, void* d_input_gate, void* d_decay_gate,
                               float* d_decay_param, float* d_initial_state, void* workspace,
                               int64_t batch, int64_t seq_len, int64_t dim, int64_t g_stride_b,
                               int64_t g_stride_t, int64_t x_stride_b, int64_t x_stride_t,
                               int64_t i_stride_b, int64_t i_stride_t, int64_t r_stride_b,
                               int64_t r_stride_t, double decay_scale, int dtype, void* stream) {
  if (bad_shape(batch, seq_len, dim)) return TILEOPS_EBADSHAPE;
  if (cu_seqlens && (batch != 1 || num_seqs < 1 || num_seqs > 0x7ffffffeLL))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || dim == 0) return TILEOPS_OK;
  if (seq_len == 0) return TILEOPS_EBADSHAPE;
  if (!dy || !x || !input_gate || !decay_gate || !decay_param || !states || !dx ||
      !d_input_gate || !d_decay_gate || !d_decay_param || !d_initial_state || !workspace)
    return TILEOPS_EINVAL;
  cudaStream_t s = as_stream(stream);
  const Strides st{x_stride_b, x_stride_t, i_stride_b, i_stride_t,
                   r_stride_b, r_stride_t, g_stride_b, g_stride_t};
  const unsigned gx = static_cast<unsigned>((dim + 127) / 128);
  const dim3 grid(gx, static_cast<unsigned>(batch));
  const int N = static_cast<int>(num_seqs);
  const float c = static_cast<float>(decay_scale);
  float* part = static_cast<float*>(workspace);
  if (cu_seqlens) glr_check_seqlens<<<1, 128, 0, s>>>(cu_seqlens, N, seq_len, device_error_ptr());
  auto go = [&](auto zero) {
    using T = decltype(zero);
    glr_bwd_simple<T><<<grid, 128, 0, s>>>(
        static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(input_gate),
        static_cast<const T*>(decay_gate), decay_param, states, initial_state, d_final_state,
        cu_seqlens, N, static_cast<T*>(dx), static_cast<T*>(d_input_gate),
        static_cast<T*>(d_decay_gate), part, d_initial_state, seq_len, dim, st, c);
    glr_dparam<<<gx, 128, 0, s>>>(part, decay_param, d_decay_param,
                                  bwd_parts(batch, seq_len, dim), dim, c);
    return launch_status();
  };
  switch (dtype) {
    case TILEOPS_DT_F32: return go(float());
    case TILEOPS_DT_F16: return go(__half());
    default: return go(__nv_bfloat16());
  }
}

extern "C" int tileops_glr_decode_fwd(const void* x, const void* input_gate,
                                      const void* decay_gate, const float* decay_param,
                                      const float* state, void* y, float* new_state, int64_t batch,
                                      int64_t dim, int64_t x_stride, int64_t i_stride,
                                      int64_t r_stride, double decay_scale, int dtype,
                                      void* stream) {
  if (bad_shape(batch, 1, dim)) return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || dim == 0) return TILEOPS_OK;
  if (!x || !input_gate || !decay_gate || !decay_param || !state || !y || !new_state)
    return TILEOPS_EINVAL;
  cudaStream_t s = as_stream(stream);
  const Strides st{x_stride, 0, i_stride, 0, r_stride, 0, 0, 0};
  const dim3 grid(static_cast<unsigned>((dim + 127) / 128), static_cast<unsigned>(batch));
  const float c = static_cast<float>(decay_scale);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    glr_decode<T><<<grid, 128, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(input_gate),
                                       static_cast<const T*>(decay_gate), decay_param, state,
                                       static_cast<T*>(y), new_state, dim, st, c);
    return launch_status();
  };
  switch (dtype) {
    case TILEOPS_DT_F32: return go(float());
    case TILEOPS_DT_F16: return go(__half());
    default: return go(__nv_bfloat16());
  }
}
