// Gated linear recurrence over channels: the backward pass.  The formulas are in
// recurrence.cu.
#include "recurrence.cuh"

namespace tileops {
namespace {

// ---- backward ----
struct BwdArgs {
  const void *dy, *x, *ig, *rg;
  const float *lam, *states, *h0, *dhT;
  const int32_t* cu;
  void *dx, *di, *dr;
  float *part, *dh0;
  int T;  // tokens; all counts of tokens fit an int (bad_shape)
  int64_t D;
  Strides st;
  int N;
  float c;
  int* err;
  Consts consts;
};

// 1 / sqrt(v), of the least normal number where v is less: finite where m = 0, and it
// enters with factors (sigma_r and k, or sigmoid(lambda)) that are 0 there.
__device__ __forceinline__ float2 rsqrt2(float2 v) {
  constexpr float kLeast = 1.17549435e-38f;
  float2 r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(fmaxf(v.x, kLeast)));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(fmaxf(v.y, kLeast)));
  return r;
}

// Gates of a lane's run and u_t = m sigma_i x.
template <typename G, bool kAllNear, typename T>
__device__ __forceinline__ void bwd_gates(const T* mine, float2 k, const Consts& c, float2* a,
                                          float2* u, float2* si, float2* sr) {
  using P = Pair<T>;
  using Word = typename P::Word;
#pragma unroll
  for (int j = 0; j < G::kRun; ++j) {
    const Word* w = reinterpret_cast<const Word*>(mine + j * G::kChans);
    si[j] = sigmoid2(P::get(w[G::kTile / 2]), c);
    sr[j] = sigmoid2(P::get(w[G::kTile]), c);
    float2 m2;
    decay2<kAllNear>(fmul2(sr[j], k), a[j], m2, c);
    u[j] = fmul2(fmul2(fmul2(m2, rsqrt2(m2)), si[j]), P::get(w[0]));
  }
}

// The gradients of one token, from G = dL/dh_t; hp is the state before it.
struct TokenGrads {
  float2 dx, di, dr, dk, back;  // dk = -d log a / d k's factor; back = a G
};
template <bool kAllNear>
__device__ __forceinline__ TokenGrads token_grads(float2 g, float2 hp, float2 x, float2 a,
                                                  float2 si, float2 sr, float2 k,
                                                  const Consts& c) {
  float2 a2, m2;
  decay2<kAllNear>(fmul2(sr, k), a2, m2, c);
  const float2 rm = rsqrt2(m2);
  TokenGrads o;
  const float2 q = fmul2(rm, si);  // sigma_i / m
  o.dx = fmul2(g, fmul2(m2, q));
  o.di = fmul2(fmul2(o.dx, x), fsub2(c.one, si));
  o.back = fmul2(a, g);
  // sigma_r before x: at a shut gate (sigma_r = 0, m = 0, q up to 2^63) x then meets a zero, where
  // x q could overflow first and leave inf * 0 = NaN for a padded token's x above 4e19.
  const float2 second = fmul2(fmul2(a, fmul2(sr, q)), x);
  o.dk = fmul2(o.back, fsub2(fmul2(sr, hp), second));
  o.dr = fmul2(fmul2(o.dk, k), fsub2(sr, c.one));
  return o;
}

// The forward kernel's walk from the last token to the first.  What is carried is
// c_t = a_t G_t, the gradient of the state before token t: G_t = dy_t + c_{t+1}, so a run
// of tokens is again a map c -> A c + H, with the decays' product and
// H = a_t (dy_t + H).  The states h are walked anew from the forward's saved ones, one a
// warp's run.  A lane takes 8 tokens: decay, state and both sigmoids of each stay in
// registers, so no element's gates are computed twice but for m.
// An element takes 79 to 82 issue slots (6 on the special-function unit): 8 x 4096 x 4096 bf16
// takes 453 us, 4.2 TB/s of its 14.125 bytes an element, 0.64 of the copy rate, with 58 to
// 63% of the issue slots used, neither of the two full.
template <typename T, typename G, int kBytes, bool kPacked, int kStages>
__global__ void __launch_bounds__(G::kWarps * 32, G::kCtas)
    glr_bwd_scan(const __grid_constant__ BwdArgs p) {
  constexpr int kRun = G::kRun, kTile = G::kTile;
  static_assert(G::kWarpRun == kSegment, "a saved state for every run of a warp");
  using P = Pair<T>;
  using Word = typename P::Word;
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
  T* ring = reinterpret_cast<T*>(dynamic_smem) + warp * (kStages * 4 * kTile);
  // Packed sequences: the state before a token that begins one, what is handed to one that ends one.
  float2* first_slot = reinterpret_cast<float2*>(dynamic_smem + warps * (kStages * 4 * kTile) * sizeof(T)) +
                       warp * (2 * kRun * 32);
  float2* last_slot = first_slot + kRun * 32;
  const int runs = (T_ + G::kWarpRun - 1) / G::kWarpRun;
  const int stride = warps * static_cast<int>(size);  // runs of a step

  // Runs are counted from the last one, q = 0; run q begins at token (runs - 1 - q) kWarpRun.
  int next = (runs - 1 - (static_cast<int>(rank) * warps + warp)) * G::kWarpRun;
  const int by = stride * G::kWarpRun;  // tokens of a step
  const T* xn = static_cast<const T*>(p.x) + b * p.st.xb + ch0 + next * p.st.xt;
  const T* in = static_cast<const T*>(p.ig) + b * p.st.ib + ch0 + next * p.st.it;
  const T* rn = static_cast<const T*>(p.rg) + b * p.st.rb + ch0 + next * p.st.rt;
  const T* gn = static_cast<const T*>(p.dy) + b * p.st.gb + ch0 + next * p.st.gt;
  auto fetch = [&](int stage) {
    if (next >= 0) {
      const int len = min(T_ - next, G::kWarpRun);
      T* to = ring + stage * (4 * kTile);
      copy_tile<G, kBytes>(to, xn, p.st.xt, len, D - ch0, lane);
      copy_tile<G, kBytes>(to + kTile, in, p.st.it, len, D - ch0, lane);
      copy_tile<G, kBytes>(to + 2 * kTile, rn, p.st.rt, len, D - ch0, lane);
      copy_tile<G, kBytes>(to + 3 * kTile, gn, p.st.gt, len, D - ch0, lane);
      xn -= by * p.st.xt;
      in -= by * p.st.it;
      rn -= by * p.st.rt;
      gn -= by * p.st.gt;
      next -= by;
    }
    copies_commit();  // a group a step, empty past the end
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(s);

  if (kPacked) {
    // The gradient of an empty sequence's state passes through.
    for (int64_t n = (rank * warps + warp) * G::kGroups + group; n < p.N;
         n += size * warps * G::kGroups)
      if (p.cu[n + 1] <= p.cu[n])
        store_state(p.dh0 + n * D + ch, load_state(p.dhT ? p.dhT + n * D + ch : nullptr, have),
                    have);
    if (blockIdx.x == 0 && warp == 0) check_seqlens(p.cu, p.N, T_, lane, p.err);
  }

  const float2 lam = load_state(p.lam + ch, have);
  const float2 k = make_float2(have > 0 ? decay_rate(lam.x, p.c) : 0.0f,
                               have > 1 ? decay_rate(lam.y, p.c) : 0.0f);
  const bool near = __all_sync(~0u, k.x < kNear && k.y < kNear);
  float2 carry = both(0.0f), dk = both(0.0f);
  if (!kPacked) carry = load_state(p.dhT ? p.dhT + b * D + ch : nullptr, have);
  ex.init(warp, warps, size, pair);

  Seqs seqs{kPacked ? p.N - 1 : 0, 0, 0};
  int par = 0, stage = 0;
  for (int base = 0; base < runs; base += stride, par ^= 1) {
    const int q = base + static_cast<int>(rank) * warps + warp;
    const bool mine_exists = q < runs;
    const int w0 = mine_exists ? (runs - 1 - q) * G::kWarpRun : 0;
    const int t0 = w0 + group * kRun;
    const int len = mine_exists ? max(0, min(T_ - t0, kRun)) : 0;
    float2 state = both(0.0f);
    uint32_t starts = 0, stops = 0;  // bit j: token j begins its sequence / ends it
    bool bounds = false;             // one of the warp's tokens does
    if (mine_exists) {
      state = load_state(p.states + (b * runs + w0 / kSegment) * D + ch, have);
      if (kPacked) {
        starts = start_bits<G>(p.cu, p.N, w0, group, lane, seqs);
        bounds = __any_sync(~0u, starts != 0) || w0 + G::kWarpRun >= T_;
        if (bounds) {
          if (len > 0)
            stops = (starts >> 1 | (t0 + len == T_ ? 1u << (len - 1) : 0u)) & ((1u << len) - 1);
          starts &= (1u << len) - 1;
          get_bounds(starts, p.h0, first_slot, p.cu, p.N, t0, D, ch, have, lane, seqs.n0);
          get_bounds(stops, p.dhT, last_slot, p.cu, p.N, t0, D, ch, have, lane, seqs.n0);
        }
      }
    }
    auto begins = [&](int j) { return kPacked && (starts >> j & 1); };
    auto ends = [&](int j) { return kPacked && (stops >> j & 1); };
    auto before_seq = [&](int j) { return first_slot[j * 32 + lane]; };
    auto after_seq = [&](int j) { return last_slot[j * 32 + lane]; };

    float2 a[kRun], hp[kRun], si[kRun], sr[kRun];
    copies_wait<kStages - 1>();
    __syncwarp();  // the tiles of this step have landed, whichever lane copied them
    const T* mine = ring + stage * (4 * kTile) + G::tile_row(group * kRun) + 2 * pair;
    if (mine_exists) {
      if (near)
        bwd_gates<G, true>(mine, k, p.consts, a, hp, si, sr);
      else
        bwd_gates<G, false>(mine, k, p.consts, a, hp, si, sr);
    }
    if (len < kRun)
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (j >= len) a[j] = both(1.0f), hp[j] = si[j] = sr[j] = both(0.0f);  // the identity
    auto word = [&](int tensor, int j) {
      return P::get(*reinterpret_cast<const Word*>(mine + tensor * kTile + j * G::kChans));
    };
    auto dy_at = [&](int j) { return j < len ? word(3, j) : both(0.0f); };

    // Maps of the run: of the states (forwards) and of what is carried (backwards).
    // `plain`: nothing begins, ends or is missing in the warp's run, so nothing is asked.
    const bool plain = !bounds && mine_exists && kBytes == 16 && ch0 + G::kChans <= D &&
                       w0 + G::kWarpRun <= T_;
    Run fwd(both(1.0f), both(0.0f)), bwd(both(1.0f), both(0.0f));
    if (plain) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) fwd = join<false>(fwd, Run(a[j], hp[j]));
      bwd.A = fwd.A;
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) bwd.H = fmul2(a[j], fadd2(word(3, j), bwd.H));
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (begins(j)) fwd = Run(both(kForget), before_seq(j));
        fwd = kPacked ? Run(fwd.A.x < 0.0f ? fwd.A : ffma2(fwd.A, a[j], both(kLeastDecay)),
                            ffma2(a[j], fwd.H, hp[j]))
                      : join<false>(fwd, Run(a[j], hp[j]));
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        if (ends(j)) bwd = Run(both(kForget), after_seq(j));
        bwd = Run(kPacked && bwd.A.x < 0.0f ? bwd.A : ffma2(bwd.A, a[j], both(kLeastDecay)),
                  fmul2(a[j], fadd2(dy_at(j), bwd.H)));
      }
    }
    const Run earlier = scan_groups<G, kPacked, false>(fwd, lane, bounds);
    const Run later = scan_groups<G, kPacked, true>(bwd, lane, bounds);
    float2 cr = ex.template before<kPacked>(bwd, bounds, group == 0, carry, par, base == 0,
                                            base + stride < runs, warp, warps, size, rank, pair);
    if (group < G::kGroups - 1)
      cr = kPacked && bounds ? apply<true>(later, cr) : apply<false>(later, cr);
    float2 h = state;
    if (group > 0)
      h = kPacked && bounds ? apply<true>(earlier, state) : apply<false>(earlier, state);
    const int64_t row0 = (b * T_ + t0) * D + ch;
    T *dxp = static_cast<T*>(p.dx) + row0, *dip = static_cast<T*>(p.di) + row0,
      *drp = static_cast<T*>(p.dr) + row0;
    // The states before each token, then the tokens' gradients from the last on.
    auto finish = [&](auto all_near, auto asks) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (asks.value && begins(j)) h = before_seq(j);
        const float2 u = hp[j];
        hp[j] = h;
        h = ffma2(a[j], h, u);
      }
      if (!asks.value) {
        dxp += (kRun - 1) * D;
        dip += (kRun - 1) * D;
        drp += (kRun - 1) * D;
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        if (asks.value && ends(j)) cr = after_seq(j);
        if (asks.value && j >= len) continue;
        const TokenGrads o = token_grads<all_near.value>(
            fadd2(word(3, j), cr), hp[j], word(0, j), a[j], si[j], sr[j], k, p.consts);
        dk = fadd2(dk, o.dk);
        cr = o.back;
        if (asks.value) {
          store_pair<T, kBytes>(dxp + j * D, o.dx, have);
          store_pair<T, kBytes>(dip + j * D, o.di, have);
          store_pair<T, kBytes>(drp + j * D, o.dr, have);
          if (begins(j)) first_slot[j * 32 + lane] = cr;
        } else {
          store_pair<T, kBytes>(dxp, o.dx, 2);
          store_pair<T, kBytes>(dip, o.di, 2);
          store_pair<T, kBytes>(drp, o.dr, 2);
          dxp -= D;
          dip -= D;
          drp -= D;
        }
      }
    };
    if (plain && near)
      finish(std::true_type(), std::false_type());
    else if (plain)
      finish(std::false_type(), std::false_type());
    else if (kPacked && near)
      finish(std::true_type(), std::true_type());
    else
      finish(std::false_type(), std::true_type());
    if (kPacked && bounds)
      put_bounds(starts, p.dh0, first_slot, p.cu, p.N, t0, D, ch, have, lane, seqs.n0);
    if (!kPacked && mine_exists && t0 == 0) store_state(p.dh0 + b * D + ch, cr, have);
    __syncwarp();  // read by every lane before they are overwritten
    fetch(stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  copies_wait<0>();

  // d k of the CTA's tokens: lane groups, then warps, in a fixed order.
#pragma unroll
  for (int off = G::kPairs; off < 32; off *= 2) {
    dk.x += __shfl_xor_sync(~0u, dk.x, off);
    dk.y += __shfl_xor_sync(~0u, dk.y, off);
  }
  __syncthreads();  // the maps have been read
  if (group == 0) ex.warp_run[0][warp][pair] = make_float4(dk.x, dk.y, 0.0f, 0.0f);
  __syncthreads();
  if (warp == 0 && group == 0) {
    float2 sum = both(0.0f);
    for (int w = 0; w < warps; ++w) {
      sum.x += ex.warp_run[0][w][pair].x;
      sum.y += ex.warp_run[0][w][pair].y;
    }
    store_state(p.part + (b * size + rank) * D + ch, sum, have);
  }
}

template <typename T, typename G, int kBytes>
int launch_bwd_geo(const BwdArgs& a, int64_t batch, cudaStream_t s, int64_t* parts) {
  constexpr int kStages = sizeof(T) == 2 ? 2 : 1;
  const ScanGrid g = scan_grid<G>(batch, a.T, a.D);
  *parts = batch * g.cluster;
  size_t smem = static_cast<size_t>(g.warps) * kStages * 4 * G::kTile * sizeof(T);
  if (a.cu) smem += static_cast<size_t>(g.warps) * 2 * G::kRun * 32 * sizeof(float2);
  return launch_scan(a.cu ? glr_bwd_scan<T, G, kBytes, true, kStages>
                          : glr_bwd_scan<T, G, kBytes, false, kStages>,
                     g, batch, smem, a, s);
}

// parts: how many partial sums of d k every channel has.
template <typename T>
int launch_bwd(const BwdArgs& a, int64_t batch, cudaStream_t s, int64_t* parts) {
  constexpr int64_t eb = sizeof(T);
  using Eight = Geo<16, 8, 8>;
  const int bytes = std::min({copy_bytes(a.dy, a.st.gb, a.st.gt, eb),
                              copy_bytes(a.x, a.st.xb, a.st.xt, eb),
                              copy_bytes(a.ig, a.st.ib, a.st.it, eb),
                              copy_bytes(a.rg, a.st.rb, a.st.rt, eb),
                              copy_bytes(a.dx, a.D, a.D, eb), copy_bytes(a.di, a.D, a.D, eb),
                              copy_bytes(a.dr, a.D, a.D, eb)});
  if (bytes == 16) {
    // One CTA of 15 warps an SM where the channels make at most one each, and at least one
    // for every second (the forward's rule; 1 x 16384 x 2048 bf16 134 us, with 8 warps 180).
    // With more channels it would gain nothing: 1 x 16384 x 2560 256 us both ways, x 4096 251
    // and 257, 1 x 1024 x 4096 32 and 34.
    const int64_t ctas = (a.D + 15) / 16 * batch, sms = sm_count();
    if (ctas <= sms && 2 * ctas > sms)
      return launch_bwd_geo<T, Geo<16, 8, 15>, 16>(a, batch, s, parts);
    return launch_bwd_geo<T, Eight, 16>(a, batch, s, parts);
  }
  if constexpr (sizeof(T) == 2) {
    if (bytes == 2) return launch_bwd_geo<T, Eight, 2>(a, batch, s, parts);
  }
  return launch_bwd_geo<T, Eight, 4>(a, batch, s, parts);
}

// dlambda = -c sigmoid(lambda) sum of the partial sums, added in a fixed order: 32 channels
// a CTA, eight threads a channel.
__global__ void __launch_bounds__(256)
    glr_dparam(const float* part, const float* lam, float* dlam, int64_t parts, int64_t D, float c) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t d = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (d < D)
#pragma unroll 4
    for (int64_t p = slice; p < parts; p += 8) s += part[p * D + d];
  red[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && d < D) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    dlam[d] = -s * c / (1.0f + expf(-lam[d]));
  }
}

}  // namespace
}  // namespace tileops

using namespace tileops;

extern "C" int64_t tileops_glr_bwd_workspace_bytes(int64_t batch, int64_t seq_len, int64_t dim) {
  if (bad_shape(batch, seq_len, dim)) return -1;
  return batch * kMaxCluster * dim * 4;  // a partial sum a CTA along the tokens
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
  if (cu_seqlens && (batch != 1 || num_seqs < 1 || num_seqs > 0x3fffffffLL))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || dim == 0) return TILEOPS_OK;
  if (seq_len == 0) return TILEOPS_EBADSHAPE;
  if (!dy || !x || !input_gate || !decay_gate || !decay_param || !states || !dx ||
      !d_input_gate || !d_decay_gate || !d_decay_param || !d_initial_state || !workspace)
    return TILEOPS_EINVAL;
  if (!aligned16(workspace)) return TILEOPS_EALIGN;
  cudaStream_t s = as_stream(stream);
  const Strides st{x_stride_b, x_stride_t, i_stride_b, i_stride_t,
                   r_stride_b, r_stride_t, g_stride_b, g_stride_t};
  const float c = static_cast<float>(decay_scale);
  float* part = static_cast<float*>(workspace);
  const BwdArgs args{dy, x, input_gate, decay_gate, decay_param, states, initial_state,
                     d_final_state, cu_seqlens, dx, d_input_gate, d_decay_gate, part,
                     d_initial_state, static_cast<int>(seq_len), dim, st, static_cast<int>(num_seqs), c,
                     cu_seqlens ? device_error_ptr() : nullptr, Consts()};
  int status;
  int64_t parts = 0;
  switch (dtype) {
    case TILEOPS_DT_F32: status = launch_bwd<float>(args, batch, s, &parts); break;
    case TILEOPS_DT_F16: status = launch_bwd<__half>(args, batch, s, &parts); break;
    default: status = launch_bwd<__nv_bfloat16>(args, batch, s, &parts);
  }
  if (status != TILEOPS_OK) return status;
  glr_dparam<<<static_cast<unsigned>((dim + 31) / 32), 256, 0, s>>>(part, decay_param,
                                                                    d_decay_param, parts, dim, c);
  return launch_status();
}

