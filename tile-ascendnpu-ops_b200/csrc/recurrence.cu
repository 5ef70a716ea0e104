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

__device__ __forceinline__ float sqrt_approx_f(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
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

// ---- vectors of channels ----
template <int Bytes> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// V channels of one token, read or written by one access.
template <typename T, int V>
struct Chans {
  using W = typename Word<V * sizeof(T)>::type;
  W w;
  __device__ __forceinline__ void load(const T* p) { w = __ldcs(reinterpret_cast<const W*>(p)); }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<W*>(p), w); }
  __device__ __forceinline__ float get(int v) const {
    T e[V];
    memcpy(e, &w, sizeof(w));
    return Cvt<T>::to_f(e[v]);
  }
  __device__ __forceinline__ void set(const float* f) {
    T e[V];
#pragma unroll
    for (int v = 0; v < V; ++v) e[v] = Cvt<T>::from_f(f[v]);
    memcpy(&w, e, sizeof(w));
  }
};

// ---- clusters: CTAs that share one channel block and split its tokens ----
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t v;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(v));
  return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes v to the place p has in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster(float2* p, uint32_t rank, float2 v) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p)), there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y)
               : "memory");
}

// ---- the scan ----
// A run of tokens is the map h -> A h + H of the state before it to the state
// after it; runs join by composition.  A run that holds the start of a packed
// sequence forgets the state before it: A = -1 says so (decays are >= 0), and
// H alone is taken, whatever the forgotten state was.
constexpr float kForget = -1.0f;

template <bool kPacked>
__device__ __forceinline__ float apply(float2 run, float h) {
  const float next = fmaf(run.x, h, run.y);
  return kPacked && run.x < 0.0f ? run.y : next;
}
template <bool kPacked>
__device__ __forceinline__ float2 join(float2 first, float2 then) {
  float2 r = make_float2(first.x * then.x, fmaf(then.x, first.y, then.y));
  if (kPacked) {
    if (first.x < 0.0f) r.x = kForget;
    if (then.x < 0.0f) r = then;
  }
  return r;
}

constexpr int kMaxWarps = 8;     // warps of a CTA
constexpr int kMaxCluster = 8;   // CTAs of a cluster

// Which of `count` tokens from t0 on start a sequence, as bits; the sequence of t0 in n0.
// Empty sequences start no token.  Every lane returns the same.
__device__ __forceinline__ uint32_t start_bits(const int32_t* cu, int N, int64_t t0, int count,
                                               int lane) {
  const int n0 = seq_of(cu, N, t0);
  uint32_t bits = cu[n0] == t0 ? 1u : 0u;
  for (int n = n0 + 1; n < N; n += 32) {
    const int64_t at = n + lane < N ? cu[n + lane] - t0 : count;
    bits |= __reduce_or_sync(~0u, at > 0 && at < count ? 1u << at : 0u);
    if (__shfl_sync(~0u, static_cast<int>(at < count), 31) == 0) break;
  }
  return bits;
}

struct FwdArgs {
  const void *x, *ig, *rg;
  const float *lam, *h0;
  const int32_t* cu;
  void* y;
  float *hT, *states;
  int64_t T, D;
  Strides st;
  int N;
  float c;
  int* err;
};

// One CTA (or cluster of CTAs) owns 32 V channels of one batch row and walks
// along its tokens; a lane owns V channels and a warp kRun tokens at a time:
//   1. load x and the gates of the run, all loads before the first use;
//   2. a_t, u_t into registers, and the run's map (A, H);
//   3. exchange the maps: between warps through shared memory, between the
//      CTAs of a cluster through distributed shared memory;
//   4. the state before the run, from the maps before it and the carried state;
//   5. the run again, token by token from that state, and the stores.
// Step 5 repeats the sequential recurrence itself, so y differs from it by the
// rounding of the state a run starts with only.  x and the gates are read once
// and y is written once.
template <typename T, int V, int kRun, bool kPacked>
__global__ void __launch_bounds__(kMaxWarps * 32) glr_fwd_scan(const FwdArgs p) {
  __shared__ float2 warp_run[2][kMaxWarps][32 * V];
  __shared__ float2 cta_run[2][kMaxCluster][32 * V];
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int warps = blockDim.x >> 5;
  const uint32_t size = cluster_size(), rank = cluster_rank();
  const int64_t b = blockIdx.y;
  const int64_t ch = static_cast<int64_t>(blockIdx.x / size) * (32 * V) + lane * V;
  const bool active = ch < p.D;
  const int64_t T_ = p.T, D = p.D;
  const T* xp = static_cast<const T*>(p.x) + b * p.st.xb + ch;
  const T* ip = static_cast<const T*>(p.ig) + b * p.st.ib + ch;
  const T* rp = static_cast<const T*>(p.rg) + b * p.st.rb + ch;
  T* yp = static_cast<T*>(p.y) + b * T_ * D + ch;
  const int64_t nseg = (T_ + kSegment - 1) / kSegment;

  if (kPacked) {
    // Sequences without a token end where they began; the offsets are checked once.
    for (int n = rank * warps + warp; n < p.N; n += size * warps)
      if (p.cu[n + 1] <= p.cu[n] && active)
        for (int v = 0; v < V; ++v)
          p.hT[n * D + ch + v] = p.h0 ? p.h0[n * D + ch + v] : 0.0f;
    if (blockIdx.x == 0 && warp == 0) {
      bool bad = false;
      for (int n = lane; n < p.N; n += 32) bad |= p.cu[n + 1] < p.cu[n];
      bad |= p.cu[0] != 0 || p.cu[p.N] != T_;
      if (bad) report_device_error(p.err, kErrBadSeqlens);
    }
  }

  float k[V], carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = active ? decay_rate(p.lam[ch + v], p.c) : 0.0f;
    carry[v] = !kPacked && active && p.h0 ? p.h0[b * D + ch + v] : 0.0f;
  }

  if (size > 1) cluster_sync();  // every CTA runs before its shared memory is written
  const int64_t stride = static_cast<int64_t>(kRun) * warps * size;
  int par = 0;
  for (int64_t base = 0; base < T_; base += stride, par ^= 1) {
    const int64_t t0 = base + static_cast<int64_t>(rank * warps + warp) * kRun;
    const int64_t left64 = T_ - t0;
    const int len = left64 >= kRun ? kRun : (left64 > 0 ? static_cast<int>(left64) : 0);
    Chans<T, V> xr[kRun], ir[kRun], rr[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (active && j < len) {
        xr[j].load(xp + (t0 + j) * p.st.xt);
        ir[j].load(ip + (t0 + j) * p.st.it);
        rr[j].load(rp + (t0 + j) * p.st.rt);
      } else {
        memset(&xr[j], 0, sizeof(xr[j]));
        memset(&ir[j], 0, sizeof(ir[j]));
        memset(&rr[j], 0, sizeof(rr[j]));
      }
    }
    // Bit j: token t0 + j starts a sequence (one bit more than the run has
    // tokens, for the end of its last one).
    uint32_t starts = 0;
    if (kPacked && len > 0) starts = start_bits(p.cu, p.N, t0, kRun + 1, lane);

    float a[kRun][V], u[kRun][V];
    float2 run[V];
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = make_float2(1.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates g = gates_of(ir[j].get(v), rr[j].get(v), k[v]);
        a[j][v] = j < len ? g.a : 1.0f;  // past the end: the identity
        u[j][v] = j < len ? sqrt_approx_f(g.m2) * g.si * xr[j].get(v) : 0.0f;
      }
      if (kPacked && (starts >> j & 1) && j < len) {
        const int64_t n = seq_of(p.cu, p.N, t0 + j);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          u[j][v] = fmaf(a[j][v], active && p.h0 ? p.h0[n * D + ch + v] : 0.0f, u[j][v]);
          a[j][v] = kForget;
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) run[v] = join<kPacked>(run[v], make_float2(a[j][v], u[j][v]));
    }

#pragma unroll
    for (int v = 0; v < V; ++v) warp_run[par][warp][lane * V + v] = run[v];
    __syncthreads();
    float h[V];
    if (size > 1) {
      // The CTA's map, to every CTA of the cluster (warp w writes to CTA w, w + warps, ...).
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float2 all = warp_run[par][0][lane * V + v];
        for (int w = 1; w < warps; ++w) all = join<kPacked>(all, warp_run[par][w][lane * V + v]);
        for (uint32_t r = warp; r < size; r += warps)
          st_cluster(&cta_run[par][rank][lane * V + v], r, all);
      }
      cluster_sync();
#pragma unroll
      for (int v = 0; v < V; ++v)
        for (uint32_t r = 0; r < size; ++r) {
          if (r == rank) h[v] = carry[v];
          carry[v] = apply<kPacked>(cta_run[par][r][lane * V + v], carry[v]);
        }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = carry[v];
#pragma unroll
      for (int v = 0; v < V; ++v)
        for (int w = 0; w < warps; ++w)
          carry[v] = apply<kPacked>(warp_run[par][w][lane * V + v], carry[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int w = 0; w < warp; ++w)
        h[v] = apply<kPacked>(warp_run[par][w][lane * V + v], h[v]);

    if (p.states && len > 0 && t0 % kSegment == 0 && active)
#pragma unroll
      for (int v = 0; v < V; ++v) p.states[(b * nseg + t0 / kSegment) * D + ch + v] = h[v];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = apply<kPacked>(make_float2(a[j][v], u[j][v]), h[v]);
      if (active && j < len) {
        Chans<T, V> o;
        o.set(h);
        o.store(yp + (t0 + j) * D);
        if (kPacked && ((starts >> (j + 1) & 1) || t0 + j + 1 == T_)) {
          const int64_t n = seq_of(p.cu, p.N, t0 + j);
#pragma unroll
          for (int v = 0; v < V; ++v) p.hT[n * D + ch + v] = h[v];
        }
      }
    }
    if (!kPacked && len > 0 && t0 + len == T_ && active)
#pragma unroll
      for (int v = 0; v < V; ++v) p.hT[b * D + ch + v] = h[v];
  }
}

// Channels per lane and the tokens' split over warps and CTAs.  V is the widest of
// one 4-byte access that every row pointer and stride allows.
struct ScanGrid {
  int warps, cluster;
  int64_t blocks;
};

inline ScanGrid scan_grid(int64_t batch, int64_t seq_len, int64_t dim, int chans, int run) {
  ScanGrid g;
  g.blocks = (dim + chans - 1) / chans;
  const int64_t runs = (seq_len + run - 1) / run;
  g.warps = static_cast<int>(std::min<int64_t>(runs, kMaxWarps));
  g.cluster = 1;
  while (g.cluster < kMaxCluster && g.blocks * batch * g.cluster < 3 * sm_count() &&
         g.cluster * g.warps < runs)
    g.cluster *= 2;
  return g;
}

template <typename K, typename A>
int launch_scan(K kernel, const ScanGrid& g, int64_t batch, const A& args, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.blocks * g.cluster), static_cast<unsigned>(batch));
  cfg.blockDim = dim3(static_cast<unsigned>(g.warps * 32));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(g.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) {
    cudaGetLastError();
    return TILEOPS_ELAUNCH;
  }
  return TILEOPS_OK;
}

// Whether rows of V elements can be read as one word: base and strides of each tensor.
inline bool rows_fit(const void* p, int64_t sb, int64_t st, int itemsize, int V) {
  return reinterpret_cast<uintptr_t>(p) % (V * itemsize) == 0 && sb % V == 0 && st % V == 0;
}

template <typename T>
int launch_fwd(const FwdArgs& a, int64_t batch, cudaStream_t s) {
  constexpr int kRun = 16, kWide = 4 / sizeof(T);
  const int eb = sizeof(T);
  const bool wide = kWide > 1 && a.D % kWide == 0 && rows_fit(a.x, a.st.xb, a.st.xt, eb, kWide) &&
                    rows_fit(a.ig, a.st.ib, a.st.it, eb, kWide) &&
                    rows_fit(a.rg, a.st.rb, a.st.rt, eb, kWide) && rows_fit(a.y, 0, 0, eb, kWide);
  const ScanGrid g = scan_grid(batch, a.T, a.D, wide ? 32 * kWide : 32, kRun);
  if (wide)
    return a.cu ? launch_scan(glr_fwd_scan<T, kWide, kRun, true>, g, batch, a, s)
                : launch_scan(glr_fwd_scan<T, kWide, kRun, false>, g, batch, a, s);
  return a.cu ? launch_scan(glr_fwd_scan<T, 1, kRun, true>, g, batch, a, s)
              : launch_scan(glr_fwd_scan<T, 1, kRun, false>, g, batch, a, s);
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
  const FwdArgs args{x, input_gate, decay_gate, decay_param, initial_state, cu_seqlens, y,
                     final_state, states, seq_len, dim, st, static_cast<int>(num_seqs),
                     static_cast<float>(decay_scale), cu_seqlens ? device_error_ptr() : nullptr};
  switch (dtype) {
    case TILEOPS_DT_F32: return launch_fwd<float>(args, batch, s);
    case TILEOPS_DT_F16: return launch_fwd<__half>(args, batch, s);
    default: return launch_fwd<__nv_bfloat16>(args, batch, s);
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
