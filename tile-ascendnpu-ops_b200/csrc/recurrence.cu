// Gated linear recurrence over channels: the forward pass and one decode step (backward:
// recurrence_bwd.cu).
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
// its limit: it enters dr and dlambda as k sigma_r / m -> sqrt(k sigma_r / 2).  1 / m stops
// at 2^63.
//
// Packed sequences (cu_seqlens): the first token of a sequence takes its
// predecessor from initial_state by selection, not by a zero factor, so
// infinities and NaN of one sequence never reach another.
#include "recurrence.cuh"

namespace tileops {
namespace {

// ---- forward ----
struct FwdArgs {
  const void *x, *ig, *rg;
  const float *lam, *h0;
  const int32_t* cu;
  void* y;
  float *hT, *states;
  int T;  // tokens; all counts of tokens fit an int (bad_shape)
  int64_t D;
  Strides st;
  int N;
  float c;
  int* err;
  Consts consts;
};

// Decays and inputs of a lane's run.
template <typename G, bool kAllNear, typename T>
__device__ __forceinline__ void fwd_run(const T* mine, float2 k, const Consts& c, float2* a,
                                        float2* u) {
  using P = Pair<T>;
  using Word = typename P::Word;
#pragma unroll
  for (int j = 0; j < G::kRun; ++j) {
    const Word* w = reinterpret_cast<const Word*>(mine + j * G::kChans);
    const float2 si = sigmoid2(P::get(w[G::kTile / 2]), c), sr = sigmoid2(P::get(w[G::kTile]), c);
    float2 m2;
    decay2<kAllNear>(fmul2(sr, k), a[j], m2, c);
    const float2 m = make_float2(sqrt_approx_f(m2.x), sqrt_approx_f(m2.y));
    u[j] = fmul2(fmul2(m, si), P::get(w[0]));
  }
}

// One CTA (or cluster of CTAs) owns 32 or 16 channels of one batch row and walks along
// its tokens; a lane owns two channels and 16 tokens of its warp's 32 or 64 at a time:
//   1. x and the gates of the run, copied to the warp's tiles a step or two ahead;
//   2. a_t, u_t into registers, and the run's map (A, H);
//   3. the maps are joined: between groups of lanes by shuffles, between warps through
//      shared memory, between the CTAs of a cluster through distributed shared memory;
//   4. so each lane has the state before its run;
//   5. the run again, token by token from that state, and the stores.
// Step 5 repeats the sequential recurrence itself, so y differs from it by the
// rounding of the state a run starts with only (infinities stay infinite as there: decays
// and their products never reach zero).  x and the gates are read once and y is
// written once.
template <typename T, typename G, int kBytes, bool kPacked, int kStages>
__global__ void __launch_bounds__(G::kWarps * 32, G::kCtas)
    glr_fwd_scan(const __grid_constant__ FwdArgs p) {
  constexpr int kRun = G::kRun, kTile = G::kTile;
  extern __shared__ __align__(16) char dynamic_smem[];
  __shared__ Exchange<G> ex;
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int warps = blockDim.x >> 5;
  const uint32_t size = cluster_size(), rank = cluster_rank();
  const int64_t b = blockIdx.y, D = p.D;
  const int T_ = p.T;
  const int group = lane / G::kPairs, pair = lane % G::kPairs;
  const int64_t ch0 = static_cast<int64_t>(blockIdx.x / size) * G::kChans, ch = ch0 + 2 * pair;
  const int have = ch + 1 < D ? 2 : (ch < D ? 1 : 0);  // channels of this lane
  T* ring = reinterpret_cast<T*>(dynamic_smem) + warp * (kStages * 3 * kTile);
  const int nseg = (T_ + kSegment - 1) / kSegment;
  const int stride = G::kWarpRun * warps * static_cast<int>(size);  // tokens of a step

  int next = (static_cast<int>(rank) * warps + warp) * G::kWarpRun;  // to be copied next
  const T* xn = static_cast<const T*>(p.x) + b * p.st.xb + ch0 + next * p.st.xt;
  const T* in = static_cast<const T*>(p.ig) + b * p.st.ib + ch0 + next * p.st.it;
  const T* rn = static_cast<const T*>(p.rg) + b * p.st.rb + ch0 + next * p.st.rt;
  auto fetch = [&](int stage) {
    if (next < T_) {
      const int len = min(T_ - next, G::kWarpRun);
      T* t = ring + stage * (3 * kTile);
      copy_tile<G, kBytes>(t, xn, p.st.xt, len, D - ch0, lane);
      copy_tile<G, kBytes>(t + kTile, in, p.st.it, len, D - ch0, lane);
      copy_tile<G, kBytes>(t + 2 * kTile, rn, p.st.rt, len, D - ch0, lane);
      xn += stride * p.st.xt;
      in += stride * p.st.it;
      rn += stride * p.st.rt;
      next += stride;
    }
    copies_commit();  // a group a step, empty past the end
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(s);

  if (kPacked) {
    // Sequences without a token end where they began.
    for (int64_t n = (rank * warps + warp) * G::kGroups + group; n < p.N;
         n += size * warps * G::kGroups)
      if (p.cu[n + 1] <= p.cu[n])
        store_state(p.hT + n * D + ch, load_state(p.h0 ? p.h0 + n * D + ch : nullptr, have), have);
    if (blockIdx.x == 0 && warp == 0) check_seqlens(p.cu, p.N, T_, lane, p.err);
  }

  const float2 lam = load_state(p.lam + ch, have);
  const float2 k = make_float2(have > 0 ? decay_rate(lam.x, p.c) : 0.0f,
                               have > 1 ? decay_rate(lam.y, p.c) : 0.0f);
  // -log a = k sigmoid(r) <= k.
  const bool near = __all_sync(~0u, k.x < kNear && k.y < kNear);
  float2 carry = both(0.0f);
  if (!kPacked) carry = load_state(p.h0 ? p.h0 + b * D + ch : nullptr, have);
  ex.init(warp, warps, size, pair);

  Seqs seqs{0, 0, 0};
  int par = 0, stage = 0;
  // (64-bit counters here: with 32-bit ones ptxas spilled 44 bytes, 214 -> 247 us.)
  for (int64_t base = 0; base < T_; base += stride, par ^= 1) {
    const int64_t w0 = base + (static_cast<int>(rank) * warps + warp) * G::kWarpRun;
    const int64_t t0 = w0 + group * kRun, left = T_ - t0;
    const int len = left >= kRun ? kRun : (left > 0 ? static_cast<int>(left) : 0);
    uint32_t starts = 0, stops = 0;  // bit j: token j begins its sequence / ends it
    bool bounds = false;             // one of the warp's tokens does
    if (kPacked && w0 < T_) {
      starts = start_bits<G>(p.cu, p.N, static_cast<int>(w0), group, lane, seqs);
      bounds = __any_sync(~0u, starts != 0) || w0 + G::kWarpRun >= T_;
      if (bounds) {
        if (len > 0)
          stops = (starts >> 1 | (t0 + len == T_ ? 1u << (len - 1) : 0u)) & ((1u << len) - 1);
        starts &= (1u << len) - 1;
      }
    }

    float2 a[kRun], u[kRun];
    copies_wait<kStages - 1>();
    __syncwarp();  // the tiles of this step have landed, whichever lane copied them
    const T* mine = ring + stage * (3 * kTile) + G::tile_row(group * kRun) + 2 * pair;
    if (w0 < T_) {
      if (near)
        fwd_run<G, true>(mine, k, p.consts, a, u);
      else
        fwd_run<G, false>(mine, k, p.consts, a, u);
    }
    __syncwarp();  // read by every lane before they are overwritten
    // A run with bounds keeps its tile a while longer, for their states.
    const int here = stage;
    float2* slot = reinterpret_cast<float2*>(ring + here * (3 * kTile));
    static_assert(3 * kTile * sizeof(T) >= kRun * 32 * sizeof(float2), "a state for every token");
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (!bounds) fetch(here);
    if (len < kRun)
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (j >= len) a[j] = both(1.0f), u[j] = both(0.0f);  // past the end: the identity
    if (kPacked && bounds) {
      get_bounds(starts, p.h0, slot, p.cu, p.N, t0, D, ch, have, lane, seqs.n0);
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (starts >> j & 1) {
          u[j] = ffma2(a[j], slot[j * 32 + lane], u[j]);
          a[j] = both(kForget);
        }
    }
    Run run = {a[0], u[0]};
    if (kPacked && bounds)
#pragma unroll
      for (int j = 1; j < kRun; ++j) run = join<true>(run, Run{a[j], u[j]});
    else
#pragma unroll
      for (int j = 1; j < kRun; ++j) run = join<false>(run, Run{a[j], u[j]});
    const Run earlier = scan_groups<G, kPacked, false>(run, lane, bounds);
    float2 h = ex.template before<kPacked>(run, bounds, group == G::kGroups - 1, carry, par, base == 0,
                                           base + stride < T_, warp, warps, size, rank, pair);
    if (group > 0) h = kPacked && bounds ? apply<true>(earlier, h) : apply<false>(earlier, h);

    if (p.states && len > 0 && t0 % kSegment == 0)
      store_state(p.states + (b * nseg + t0 / kSegment) * D + ch, h, have);
    T* yp = static_cast<T*>(p.y) + (b * T_ + t0) * D + ch;
    if (!bounds && kBytes == 16 && len == kRun && ch0 + G::kChans <= D) {
#pragma unroll
      for (int j = 0; j < kRun; ++j, yp += D) {
        h = apply<false>(Run{a[j], u[j]}, h);
        store_pair<T, kBytes>(yp, h, 2);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        h = apply<kPacked>(Run{a[j], u[j]}, h);
        if (j < len) {
          store_pair<T, kBytes>(yp + j * D, h, have);
          if (kPacked && (stops >> j & 1)) slot[j * 32 + lane] = h;
        }
      }
    }
    if (kPacked && bounds) {
      put_bounds(stops, p.hT, slot, p.cu, p.N, t0, D, ch, have, lane, seqs.n0);
      __syncwarp();
      fetch(here);
    }
    if (!kPacked && len > 0 && t0 + len == T_) store_state(p.hT + b * D + ch, h, have);
  }
  copies_wait<0>();
}

template <typename T, typename G, int kBytes, int kStages>
int launch_fwd_geo(const FwdArgs& a, int64_t batch, cudaStream_t s) {
  const ScanGrid g = scan_grid<G>(batch, a.T, a.D);
  const size_t smem = static_cast<size_t>(g.warps) * kStages * 3 * G::kTile * sizeof(T);
  return launch_scan(a.cu ? glr_fwd_scan<T, G, kBytes, true, kStages>
                          : glr_fwd_scan<T, G, kBytes, false, kStages>,
                     g, batch, smem, a, s);
}

template <typename T>
int launch_fwd(const FwdArgs& a, int64_t batch, cudaStream_t s) {
  constexpr int kStages = sizeof(T) == 2 ? 2 : 1;  // about 100 KB of tiles: two CTAs an SM
  constexpr int64_t eb = sizeof(T);
  using Wide = Geo<32, 16, 8>;
  const int bytes = std::min({copy_bytes(a.x, a.st.xb, a.st.xt, eb),
                              copy_bytes(a.ig, a.st.ib, a.st.it, eb),
                              copy_bytes(a.rg, a.st.rb, a.st.rt, eb),
                              copy_bytes(a.y, a.D, a.D, eb)});
  if (bytes == 16) {
    // More CTAs than SMs: two of 8 warps an SM.  Fewer: one of 15 warps that has the SM for
    // itself, of 16 channels (more copies and shuffles an element) where those of 32
    // would leave half the SMs idle.  Fewer still: two of 8 warps an SM in
    // clusters, as one waits for its cluster while the other computes.
    // 1 x 16384 x D bf16: D = 4096 120 us, with 8 warps and 16 channels 147; 2048 72 us,
    // with 8 warps 83; 1024 55 us in clusters, with 15 warps 73; 256 28 and 48.  Above the
    // first bound: 5120 236 us, with 15 warps 235; 1 x 1024 x 5120 21 us and 27.
    const int64_t ctas = (a.D + 31) / 32 * batch, sms = sm_count();
    if (ctas > sms) return launch_fwd_geo<T, Wide, 16, kStages>(a, batch, s);
    if (2 * ctas > sms) return launch_fwd_geo<T, Geo<32, 16, 15>, 16, kStages>(a, batch, s);
    if (4 * ctas > sms) return launch_fwd_geo<T, Geo<16, 16, 15>, 16, kStages>(a, batch, s);
    return launch_fwd_geo<T, Geo<16, 16, 8>, 16, kStages>(a, batch, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (bytes == 2) return launch_fwd_geo<T, Wide, 2, kStages>(a, batch, s);
  }
  return launch_fwd_geo<T, Geo<16, 16, 8>, 4, kStages>(a, batch, s);
}

// ---- one token ----
// Four channels a thread where every row starts on the boundary of four (kVec = 4), one
// otherwise.  A thread reads all it needs before it writes, so hn may be h0.
template <typename T, int kVec>
__global__ void __launch_bounds__(128)
    glr_decode(const T* x, const T* ig, const T* rg, const float* lam, const float* h0, T* y,
               float* hn, int64_t D, Strides st, float c) {
  const int64_t d = (blockIdx.x * 128ll + threadIdx.x) * kVec, b = blockIdx.y;
  if (d >= D) return;
  T xv[kVec], iv[kVec], rv[kVec], yv[kVec];
  float lv[kVec], hv[kVec];
  auto load = [](auto* to, const auto* from) {
    if constexpr (kVec == 1) {
      *to = *from;
    } else {
      struct alignas(kVec * sizeof(*to)) Words {
        uint32_t w[kVec * sizeof(*to) / 4];
      };
      const Words words = *reinterpret_cast<const Words*>(from);
      memcpy(to, &words, sizeof(words));
    }
  };
  auto store = [](auto* to, const auto* from) {
    if constexpr (kVec == 1) {
      *to = *from;
    } else {
      struct alignas(kVec * sizeof(*to)) Words {
        uint32_t w[kVec * sizeof(*to) / 4];
      };
      Words words;
      memcpy(&words, from, sizeof(words));
      *reinterpret_cast<Words*>(to) = words;
    }
  };
  load(lv, lam + d);
  load(hv, h0 + b * D + d);
  load(iv, ig + b * st.ib + d);
  load(rv, rg + b * st.rb + d);
  load(xv, x + b * st.xb + d);
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const Gates g = gates_of(Cvt<T>::to_f(iv[v]), Cvt<T>::to_f(rv[v]), decay_rate(lv[v], c));
    hv[v] = fmaf(g.a, hv[v], sqrt_approx_f(g.m2) * g.si * Cvt<T>::to_f(xv[v]));
    yv[v] = Cvt<T>::from_f(hv[v]);
  }
  store(y + b * D + d, yv);
  store(hn + b * D + d, hv);
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
  if (cu_seqlens && (batch != 1 || num_seqs < 1 || num_seqs > 0x3fffffffLL))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || dim == 0) return TILEOPS_OK;
  if (seq_len == 0) return TILEOPS_EBADSHAPE;
  if (!x || !input_gate || !decay_gate || !decay_param || !y || !final_state)
    return TILEOPS_EINVAL;
  cudaStream_t s = as_stream(stream);
  const Strides st{x_stride_b, x_stride_t, i_stride_b, i_stride_t, r_stride_b, r_stride_t, 0, 0};
  const FwdArgs args{x, input_gate, decay_gate, decay_param, initial_state, cu_seqlens, y,
                     final_state, states, static_cast<int>(seq_len), dim, st, static_cast<int>(num_seqs),
                     static_cast<float>(decay_scale), cu_seqlens ? device_error_ptr() : nullptr, Consts()};
  switch (dtype) {
    case TILEOPS_DT_F32: return launch_fwd<float>(args, batch, s);
    case TILEOPS_DT_F16: return launch_fwd<__half>(args, batch, s);
    default: return launch_fwd<__nv_bfloat16>(args, batch, s);
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
  const float c = static_cast<float>(decay_scale);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    auto fits = [](const void* p, int64_t stride, size_t itemsize) {
      return reinterpret_cast<uintptr_t>(p) % (4 * itemsize) == 0 && stride % 4 == 0;
    };
    const bool vec = fits(x, x_stride, sizeof(T)) && fits(input_gate, i_stride, sizeof(T)) &&
                     fits(decay_gate, r_stride, sizeof(T)) && fits(y, dim, sizeof(T)) &&
                     fits(state, dim, 4) && fits(new_state, dim, 4) && fits(decay_param, 4, 4);
    const int64_t per_cta = vec ? 512 : 128;
    const dim3 grid(static_cast<unsigned>((dim + per_cta - 1) / per_cta),
                    static_cast<unsigned>(batch));
    auto kernel = vec ? glr_decode<T, 4> : glr_decode<T, 1>;
    kernel<<<grid, 128, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(input_gate),
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
