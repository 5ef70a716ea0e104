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
#include <type_traits>

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

// a and 1 - a^2 from f = -log a >= 0.  Near zero both come from g = 1 - a = 1 - exp(-f):
// 1 - a^2 = g (1 + a) has no cancellation, and a = 1 - g rounds once, where an approximate
// exponential's error would be carried along the whole sequence.  g / f on [0, 1/4] is a
// polynomial of degree 4 fitted here by Remez exchange on the relative error: 8e-9 with
// its coefficients in fp32, a seventh of half a step.
constexpr float kNear = 0.25f;
constexpr float kG0 = 1.0f, kG1 = -0.4999994933605194f, kG2 = 0.16665081679821014f,
                kG3 = -0.041488952934741974f, kG4 = 0.007510221563279629f;

__device__ __forceinline__ void decay_of(float f, float& a, float& m2) {
  float p = fmaf(f, kG4, kG3);
  p = fmaf(f, p, kG2);
  p = fmaf(f, p, kG1);
  p = fmaf(f, p, kG0);
  const float g = f * p;
  const float e = ex2_approx_f(-kLog2e * f);
  const bool near = f < kNear;
  a = near ? 1.0f - g : e;
  m2 = near ? g * (1.0f + a) : fmaf(-e, e, 1.0f);
}

__device__ __forceinline__ Gates gates_of(float i, float r, float k) {
  Gates g;
  g.si = sigmoid_f(i);
  g.sr = sigmoid_f(r);
  decay_of(k * g.sr, g.a, g.m2);
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
// The sequence token t belongs to, the last n with cu[n] <= t, in [0, N); from a guess
// nearby: doubling steps away from it, then halves.
__device__ __forceinline__ int seq_near(const int32_t* cu, int N, int t, int guess) {
  int lo = guess, hi = guess + 1;
  if (cu[guess] <= t) {
    for (int by = 1; hi < N && cu[hi] <= t; by *= 2) {
      lo = hi;
      hi = N - hi < by ? N : hi + by;
    }
  } else {
    hi = guess;
    for (int by = 1; lo > 0 && cu[lo] > t; by *= 2) {
      hi = lo;
      lo = lo < by ? 0 : lo - by;
    }
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

struct Strides {
  int64_t xb, xt, ib, it, rb, rt, gb, gt;  // x, input gate, decay gate, dy: batch and token
};

// ---- two channels at a time ----
// The kernels below give a lane two neighbouring channels: their arithmetic is
// packed (fma.rn.f32x2 and its kin, one issue slot for both).
__device__ __forceinline__ float2 fsub2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "sub.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <typename T>
struct Pair;  // two values of T as they lie in memory
template <>
struct Pair<float> {
  using Word = uint2;
  static __device__ __forceinline__ float2 get(Word w) {
    return make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
  }
  static __device__ __forceinline__ Word set(float2 v) {
    return make_uint2(__float_as_uint(v.x), __float_as_uint(v.y));
  }
};
template <>
struct Pair<__nv_bfloat16> {
  using Word = uint32_t;
  static __device__ __forceinline__ float2 get(Word w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ Word set(float2 v) {
    const __nv_bfloat162 r = __float22bfloat162_rn(v);
    Word w;
    memcpy(&w, &r, 4);
    return w;
  }
};
template <>
struct Pair<__half> {
  using Word = uint32_t;
  static __device__ __forceinline__ float2 get(Word w) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
  }
  static __device__ __forceinline__ Word set(float2 v) {
    const __half2 r = __float22half2_rn(v);
    Word w;
    memcpy(&w, &r, 4);
    return w;
  }
};

// Constants of the packed arithmetic, handed over as kernel arguments: from there
// they go to uniform registers, where literals would take a register pair each.
struct Consts {
  float2 nlog2e = {-kLog2e, -kLog2e}, one = {1.0f, 1.0f}, g1 = {kG1, kG1}, g2 = {kG2, kG2},
         g3 = {kG3, kG3}, g4 = {kG4, kG4};
};

__device__ __forceinline__ float2 sigmoid2(float2 z, const Consts& c) {
  const float2 t = fmul2(z, c.nlog2e);
  const float2 d = fadd2(make_float2(ex2_approx_f(t.x), ex2_approx_f(t.y)), c.one);
  return make_float2(rcp_approx_f(d.x), rcp_approx_f(d.y));
}

// decay_of of two channels; kAllNear: both are known to be near zero.
template <bool kAllNear>
__device__ __forceinline__ void decay2(float2 f, float2& a, float2& m2, const Consts& c) {
  float2 p = ffma2(f, c.g4, c.g3);
  p = ffma2(f, p, c.g2);
  p = ffma2(f, p, c.g1);
  p = ffma2(f, p, c.one);
  const float2 g = fmul2(f, p);
  a = fsub2(c.one, g);
  m2 = fmul2(g, fadd2(a, c.one));
  if (!kAllNear) {
    const float2 t = fmul2(f, c.nlog2e);
    const float2 e = make_float2(ex2_approx_f(t.x), ex2_approx_f(t.y));
    const float2 o = fsub2(c.one, fmul2(e, e));
    if (!(f.x < kNear)) a.x = e.x, m2.x = o.x;
    if (!(f.y < kNear)) a.y = e.y, m2.y = o.y;
  }
}

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
__device__ __forceinline__ void st_cluster(float4* p, uint32_t rank, float4 v) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p)), there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// ---- the scan ----
// A run of tokens is the map h -> A h + H of the state before it to the state
// after it; runs join by composition.  A run that holds the start of a packed
// sequence forgets the state before it: A = -1 says so (decays are >= 0), and
// H alone is taken, whatever the forgotten state was.
constexpr float kForget = -1.0f;

struct Run {
  float2 A, H;  // of two channels
  __device__ __forceinline__ Run(float2 a, float2 h) : A(a), H(h) {}
  __device__ __forceinline__ explicit Run(float4 w)
      : A(make_float2(w.x, w.y)), H(make_float2(w.z, w.w)) {}
  __device__ __forceinline__ float4 word() const { return make_float4(A.x, A.y, H.x, H.y); }
};

// The map of the lane `by` below (backwards: above).
template <bool kBackwards>
__device__ __forceinline__ Run shuffle_by(const Run& r, int by) {
  auto f = [&](float v) {
    return kBackwards ? __shfl_down_sync(~0u, v, by) : __shfl_up_sync(~0u, v, by);
  };
  return Run(make_float2(f(r.A.x), f(r.A.y)), make_float2(f(r.H.x), f(r.H.y)));
}

template <bool kPacked>
__device__ __forceinline__ float2 apply(const Run& run, float2 h) {
  float2 next = ffma2(run.A, h, run.H);
  if (kPacked) {
    if (run.A.x < 0.0f) next.x = run.H.x;
    if (run.A.y < 0.0f) next.y = run.H.y;
  }
  return next;
}
template <bool kPacked>
__device__ __forceinline__ Run join(const Run& first, const Run& then) {
  Run r(fmul2(first.A, then.A), apply<kPacked>(then, first.H));
  if (kPacked) {
    if (first.A.x < 0.0f || then.A.x < 0.0f) r.A.x = kForget;
    if (first.A.y < 0.0f || then.A.y < 0.0f) r.A.y = kForget;
  }
  return r;
}

constexpr int kMaxWarps = 8;    // warps of a CTA
constexpr int kMaxCluster = 8;  // CTAs of a cluster

// How a warp lies over channels and tokens: `Chans` channels side by side, two a lane,
// and groups of lanes one after another in time, `Run` tokens a lane.
template <int Chans, int Run>
struct Geo {
  static constexpr int kChans = Chans, kRun = Run;
  static constexpr int kPairs = Chans / 2, kGroups = 32 / kPairs;
  static constexpr int kWarpRun = Run * kGroups;                // tokens of a warp
  static constexpr int kTile = (kWarpRun + kGroups) * Chans;    // elements of its tile
  static __device__ __forceinline__ constexpr int tile_row(int row) {
    return (row + row / Run) * Chans;
  }
};

// ---- a warp's rows in shared memory ----
// A tile is kWarpRun tokens of the channels of the warp, rows of one tensor one
// below another, a row left out after each group's so that the groups read
// different banks.  The warp copies its own tiles and only it reads them, so no
// barrier but its own is needed.  kBytes: what one copy moves, the widest that
// the tensors' addresses and strides allow (16; 4; 2 by plain loads, as
// cp.async has no such size).
__device__ __forceinline__ void copy16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(in ? 16 : 0)
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

// Copies `len` rows (0 < len <= kWarpRun) starting at `row0`, which points at the first
// of the CTA's channels; `left` of them exist (0 < left).  What does not exist
// is filled with zeros and not read: its source is `row0` itself.
template <typename G, int kBytes, typename T>
__device__ __forceinline__ void copy_tile(T* tile, const T* row0, int64_t stride, int len,
                                          int64_t left, int lane) {
  constexpr int kEach = kBytes / sizeof(T);   // elements of one copy
  constexpr int kPerRow = G::kChans / kEach;     // copies of a row
  constexpr int kRows = 32 / kPerRow;         // rows of one instruction
  static_assert(32 % kPerRow == 0 && (kRows % G::kRun == 0 || G::kRun % kRows == 0), "copies of a row");
  const int r0 = lane / kPerRow, col = lane % kPerRow * kEach;
  const T* src = row0 + r0 * stride + col;
  if (kBytes == 16 && len == G::kWarpRun && left >= G::kChans) {
#pragma unroll
    for (int i = 0; i < G::kWarpRun / kRows; ++i, src += kRows * stride)
      copy16(tile + G::tile_row(i * kRows + r0) + col, src, true);
    return;
  }
#pragma unroll
  for (int i = 0; i < G::kWarpRun / kRows; ++i, src += kRows * stride) {
    const bool in = i * kRows + r0 < len && col < left;
    T* dst = tile + G::tile_row(i * kRows + r0) + col;
    if constexpr (kBytes == 16)
      copy16(dst, in ? src : row0, in);
    else if constexpr (kBytes == 4)
      copy4(dst, in ? src : row0, in);
    else
      *dst = in ? *src : Cvt<T>::from_f(0.0f);
  }
}

// Stores two neighbouring channels; kBytes < the pair's size: one by one.
template <typename T, int kBytes>
__device__ __forceinline__ void store_pair(T* p, float2 v, int have) {
  if constexpr (kBytes >= 2 * sizeof(T)) {
    if (have > 0)
      __stcs(reinterpret_cast<typename Pair<T>::Word*>(p), Pair<T>::set(v));
  } else {
    if (have > 0) p[0] = Cvt<T>::from_f(v.x);
    if (have > 1) p[1] = Cvt<T>::from_f(v.y);
  }
}
__device__ __forceinline__ float2 load_state(const float* p, int have) {
  return make_float2(p && have > 0 ? p[0] : 0.0f, p && have > 1 ? p[1] : 0.0f);
}
__device__ __forceinline__ void store_state(float* p, float2 v, int have) {
  if (have > 0) p[0] = v.x;
  if (have > 1) p[1] = v.y;
}

// Where a warp is among the packed sequences, the same in all lanes.
struct Seqs {
  int n0;      // the sequence of the run's first token w0
  int lo, hi;  // its bounds
};

// Which tokens of a lane's run start a sequence: bit j for token t0 + j, j = 0 .. kRun (one
// more than the run has, for the end of its last token).  Empty sequences start
// no token.  w0: the first token of the warp's run, the same in every lane.  A
// run strictly inside the sequence found last needs no search; one that is not
// costs two loads by the whole warp where the next sequence is near.
template <typename G>
__device__ __forceinline__ uint32_t start_bits(const int32_t* cu, int N, int w0, int group,
                                               int lane, Seqs& s) {
  static_assert(G::kWarpRun <= 64, "bits of a warp's run");
  if (s.lo < w0 && w0 + G::kWarpRun < s.hi) return 0;
  if (cu[s.n0] <= w0) {
    for (;;) {  // forwards: entries after n0 that are <= w0
      const int n = s.n0 + 1 + lane;
      const uint32_t past = __ballot_sync(~0u, n < N && cu[n] <= w0);
      s.n0 += __popc(past);
      if (past != ~0u) break;
    }
  } else {
    for (;;) {  // backwards: the nearest entry <= w0 (the first one if there is none)
      const int n = s.n0 - lane;
      const uint32_t found = __ballot_sync(~0u, n <= 0 || cu[n] <= w0);
      s.n0 = max(0, s.n0 - (found ? __ffs(found) - 1 : 32));
      if (found) break;
    }
  }
  s.lo = cu[s.n0];
  s.hi = cu[s.n0 + 1];
  uint64_t bits = s.lo == w0 ? 1 : 0;
  uint32_t beyond = 0;  // token w0 + 64
  for (int n = s.n0 + 1;; n += 32) {
    const int64_t far = n + lane < N ? int64_t{cu[n + lane]} - w0 : G::kWarpRun + 1;
    const int at = static_cast<int>(min(max(far, int64_t{-1}), int64_t{G::kWarpRun + 1}));
    const uint64_t mine = at > 0 && at < 64 ? 1ull << at : 0ull;
    bits |= static_cast<uint64_t>(__reduce_or_sync(~0u, static_cast<uint32_t>(mine >> 32))) << 32 |
            __reduce_or_sync(~0u, static_cast<uint32_t>(mine));
    beyond |= __any_sync(~0u, at == 64);
    if (n + 32 >= N || __shfl_sync(~0u, static_cast<int>(at <= G::kWarpRun), 31) == 0) break;
  }
  uint32_t run = static_cast<uint32_t>(bits >> (group * G::kRun)) & ((1u << (G::kRun + 1)) - 1);
  if (group * G::kRun + G::kRun == 64) run |= beyond << G::kRun;
  return run;
}

// For each token of `bits` (of the lane's run), v of its sequence into slot[token][lane].
// Rolled on purpose, like put_bounds: unrolled over the tokens the searches made the kernels
// miss the instruction cache (5 us a bound).
__device__ __forceinline__ void get_bounds(uint32_t bits, const float* v, float2* slot,
                                           const int32_t* cu, int N, int t0, int64_t D,
                                           int64_t ch, int have, int lane, int n0) {
#pragma unroll 1
  for (; bits; bits &= bits - 1) {
    const int j = __ffs(bits) - 1;
    const int64_t n = seq_near(cu, N, t0 + j, n0);
    slot[j * 32 + lane] = load_state(v ? v + n * D + ch : nullptr, have);
  }
}
// The reverse: slot[token][lane] to v of the token's sequence.
__device__ __forceinline__ void put_bounds(uint32_t bits, float* v, const float2* slot,
                                           const int32_t* cu, int N, int t0, int64_t D,
                                           int64_t ch, int have, int lane, int n0) {
#pragma unroll 1
  for (; bits; bits &= bits - 1) {
    const int j = __ffs(bits) - 1;
    const int64_t n = seq_near(cu, N, t0 + j, n0);
    store_state(v + n * D + ch, slot[j * 32 + lane], have);
  }
}

// Warp w passes on to the next one, which waits: hardware barrier 1 + w counts
// the 32 threads of each.  A warp passes a second time only after the state has
// gone all the way round, so its successor has long waited for the first.
__device__ __forceinline__ void link_pass(int w) {
  asm volatile("bar.arrive %0, 64;" ::"r"(1 + w) : "memory");
}
__device__ __forceinline__ void link_wait(int w) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + w) : "memory");
}

// Joins the maps of a warp's lane groups in their order (backwards: from the last): `run`
// comes back as the map up to and with the lane's own, and the result is the
// one up to its predecessor (of no meaning in the first group).  bounds: the
// warp's run has tokens that forget.
template <typename G, bool kPacked, bool kBackwards>
__device__ __forceinline__ Run scan_groups(Run& run, int lane, bool bounds) {
#pragma unroll
  for (int off = G::kPairs; off < 32; off *= 2) {
    const Run other = shuffle_by<kBackwards>(run, off);
    const Run longer = kPacked && bounds ? join<true>(other, run) : join<false>(other, run);
    if (kBackwards ? lane + off < 32 : lane >= off) run = longer;
  }
  return shuffle_by<kBackwards>(run, G::kPairs);
}

// ---- the state before a warp's run ----
// Warps take their runs in the order of the scan: q = step * warps * size + rank * warps
// + warp (size CTAs of a cluster, this one `rank`).
template <typename G>
struct Exchange {
  float4 warp_run[2][kMaxWarps][G::kPairs];  // (A, H) of two channels
  float4 cta_run[2][kMaxCluster][G::kPairs];

  // Maps of warps and CTAs that do not exist stay the identity.
  __device__ __forceinline__ void init(int warp, int warps, uint32_t size, int pair) {
    const float4 identity = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
    for (int w = warp; w < kMaxWarps; w += warps)
      warp_run[0][w][pair] = warp_run[1][w][pair] = identity;
    for (int r = warp; r < kMaxCluster; r += warps)
      cta_run[0][r][pair] = cta_run[1][r][pair] = identity;
    __syncthreads();
    if (size > 1) cluster_sync();  // every CTA got here before another writes its maps
  }

  // `run`: the map of the whole warp's run, in the lanes of `holder`.  carry: the state
  // before the step (a cluster) or before everything (one CTA).  Two buffers in turn:
  // one is written again only after a barrier that every reader has passed.
  template <bool kPacked>
  __device__ __forceinline__ float2 before(const Run& run, bool bounds, bool holder, float2& carry, int par,
                                           bool first, bool more, int warp, int warps,
                                           uint32_t size, uint32_t rank, int pair) {
    float2 h = carry;
    if (size > 1) {
      if (holder) warp_run[par][warp][pair] = run.word();
      __syncthreads();
      // The CTA's map, to every CTA of the cluster (warp w writes to CTA w, w + warps, ...).
      Run all(warp_run[par][0][pair]);
#pragma unroll
      for (int w = 1; w < kMaxWarps; ++w)
        all = join<kPacked>(all, Run(warp_run[par][w][pair]));
      if (holder)
        for (uint32_t r = warp; r < size; r += warps)
          st_cluster(&cta_run[par][rank][pair], r, all.word());
      __syncwarp();
      cluster_sync();
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r) {
        if (r == rank) h = carry;
        carry = apply<kPacked>(Run(cta_run[par][r][pair]), carry);
      }
#pragma unroll
      for (int w = 0; w < kMaxWarps - 1; ++w)
        if (w < warp) h = apply<kPacked>(Run(warp_run[par][w][pair]), h);
    } else {
      // A chain from warp to warp: the state goes on as soon as it is known, and
      // each warp waits for its predecessor alone.
      float4* link = warp_run[0][0];  // [warp][pair]: the state before a warp's run
      if (!first || warp > 0) {
        if (warps > 1)
          link_wait(warp == 0 ? warps - 1 : warp - 1);
        else
          __syncwarp();
        const float4 v = link[warp * G::kPairs + pair];
        h = make_float2(v.x, v.y);
      }
      if (more || warp + 1 < warps) {
        const int to = warp + 1 == warps ? 0 : warp + 1;
        const float2 out = kPacked && bounds ? apply<true>(run, h) : apply<false>(run, h);
        if (warps == 1) __syncwarp();  // read above before it is overwritten
        if (holder) link[to * G::kPairs + pair] = make_float4(out.x, out.y, 0.0f, 0.0f);
        __syncwarp();
        if (warps > 1) link_pass(warp);
      }
    }
    return h;
  }
};

// cu_seqlens must be 0 = cu[0] <= ... <= cu[N] = total; reported otherwise.
__device__ __forceinline__ void check_seqlens(const int32_t* cu, int N, int total, int lane,
                                              int* err) {
  bool bad = false;
  for (int n = lane; n < N; n += 32) bad |= cu[n + 1] < cu[n];
  bad |= cu[0] != 0 || cu[N] != total;
  if (bad) report_device_error(err, kErrBadSeqlens);
}

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
// rounding of the state a run starts with only.  x and the gates are read once
// and y is written once.
template <typename T, typename G, int kBytes, bool kPacked, int kStages>
__global__ void __launch_bounds__(kMaxWarps * 32, 2)
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
  const float2 sx = fmul2(si, x);                       // sigma_i x
  o.dx = fmul2(g, fmul2(fmul2(m2, rm), si));
  o.di = fmul2(fmul2(o.dx, x), fsub2(c.one, si));
  o.back = fmul2(a, g);
  const float2 dla = fmul2(o.back, fsub2(hp, fmul2(fmul2(a, sx), rm)));
  o.dk = fmul2(sr, dla);
  o.dr = fmul2(fmul2(o.dk, k), fsub2(sr, c.one));
  return o;
}

// The forward kernel's walk from the last token to the first.  What is carried is
// c_t = a_t G_t, the gradient of the state before token t: G_t = dy_t + c_{t+1}, so a run
// of tokens is again a map c -> A c + H, with the decays' product and
// H = a_t (dy_t + H).  The states h are walked anew from the forward's saved ones, one a
// warp's run.  A lane takes 8 tokens: decay, state and both sigmoids of each stay in
// registers, so no element's gates are computed twice but for m.
template <typename T, typename G, int kBytes, bool kPacked, int kStages>
__global__ void __launch_bounds__(kMaxWarps * 32, 2)
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
        fwd = kPacked ? Run(fwd.A.x < 0.0f ? fwd.A : fmul2(fwd.A, a[j]), ffma2(a[j], fwd.H, hp[j]))
                      : join<false>(fwd, Run(a[j], hp[j]));
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        if (ends(j)) bwd = Run(both(kForget), after_seq(j));
        bwd = Run(kPacked && bwd.A.x < 0.0f ? bwd.A : fmul2(bwd.A, a[j]),
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

// ---- launches ----
// The tokens' split over warps and CTAs: a run a warp, up to kMaxWarps; then clusters of
// 2, 4 or 8 CTAs along the tokens while the channels and batch rows alone give fewer
// CTAs than there are SMs.
struct ScanGrid {
  int warps, cluster;
  int64_t blocks;
};

template <typename G>
ScanGrid scan_grid(int64_t batch, int64_t seq_len, int64_t dim) {
  ScanGrid g;
  g.blocks = (dim + G::kChans - 1) / G::kChans;
  const int64_t runs = (seq_len + G::kWarpRun - 1) / G::kWarpRun;
  g.warps = static_cast<int>(std::min<int64_t>(runs, kMaxWarps));
  g.cluster = 1;
  while (g.cluster < kMaxCluster && g.blocks * batch * g.cluster < sm_count() &&
         g.cluster * g.warps < runs)
    g.cluster *= 2;
  return g;
}

template <typename A>
int launch_scan(void (*kernel)(const A), const ScanGrid& g, int64_t batch, size_t smem,
                const A& args, cudaStream_t s) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return TILEOPS_ELAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.blocks * g.cluster), static_cast<unsigned>(batch));
  cfg.blockDim = dim3(static_cast<unsigned>(g.warps * 32));
  cfg.dynamicSmemBytes = smem;
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

// The widest copy (16, 4 or 2 bytes) that a tensor's base and strides allow.
inline int copy_bytes(const void* p, int64_t sb, int64_t st, int64_t itemsize) {
  for (int bytes : {16, 4})
    if (reinterpret_cast<uintptr_t>(p) % bytes == 0 && sb * itemsize % bytes == 0 &&
        st * itemsize % bytes == 0)
      return bytes;
  return 2;
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
  using Wide = Geo<32, 16>;
  using Narrow = Geo<16, 16>;
  const int bytes = std::min({copy_bytes(a.x, a.st.xb, a.st.xt, eb),
                              copy_bytes(a.ig, a.st.ib, a.st.it, eb),
                              copy_bytes(a.rg, a.st.rb, a.st.rt, eb),
                              copy_bytes(a.y, a.D, a.D, eb)});
  // Sixteen channels a CTA cost more copies and shuffles an element (8 x 4096 x 4096 bf16:
  // 266 us against 233 us), but make twice the CTAs: 1 x 16384 x 4096 149 us against 159 us.
  const bool few = (a.D + 31) / 32 * batch < 2 * sm_count();
  if (bytes == 16)
    return few ? launch_fwd_geo<T, Narrow, 16, kStages>(a, batch, s)
               : launch_fwd_geo<T, Wide, 16, kStages>(a, batch, s);
  if constexpr (sizeof(T) == 2) {
    if (bytes == 2) return launch_fwd_geo<T, Wide, 2, kStages>(a, batch, s);
  }
  return launch_fwd_geo<T, Narrow, 4, kStages>(a, batch, s);
}

using BwdGeo = Geo<16, 8>;

template <typename T, int kBytes>
int launch_bwd_bytes(const BwdArgs& a, int64_t batch, cudaStream_t s) {
  constexpr int kStages = sizeof(T) == 2 ? 2 : 1;
  const ScanGrid g = scan_grid<BwdGeo>(batch, a.T, a.D);
  size_t smem = static_cast<size_t>(g.warps) * kStages * 4 * BwdGeo::kTile * sizeof(T);
  if (a.cu) smem += static_cast<size_t>(g.warps) * 2 * BwdGeo::kRun * 32 * sizeof(float2);
  return launch_scan(a.cu ? glr_bwd_scan<T, BwdGeo, kBytes, true, kStages>
                          : glr_bwd_scan<T, BwdGeo, kBytes, false, kStages>,
                     g, batch, smem, a, s);
}

template <typename T>
int launch_bwd(const BwdArgs& a, int64_t batch, cudaStream_t s) {
  constexpr int64_t eb = sizeof(T);
  const int bytes = std::min({copy_bytes(a.dy, a.st.gb, a.st.gt, eb),
                              copy_bytes(a.x, a.st.xb, a.st.xt, eb),
                              copy_bytes(a.ig, a.st.ib, a.st.it, eb),
                              copy_bytes(a.rg, a.st.rb, a.st.rt, eb),
                              copy_bytes(a.dx, a.D, a.D, eb), copy_bytes(a.di, a.D, a.D, eb),
                              copy_bytes(a.dr, a.D, a.D, eb)});
  if (bytes == 16) return launch_bwd_bytes<T, 16>(a, batch, s);
  if constexpr (sizeof(T) == 2) {
    if (bytes == 2) return launch_bwd_bytes<T, 2>(a, batch, s);
  }
  return launch_bwd_bytes<T, 4>(a, batch, s);
}

// dlambda = c sigmoid(lambda) sum of the partial sums, added in a fixed order.
__global__ void __launch_bounds__(128)
    glr_dparam(const float* part, const float* lam, float* dlam, int64_t parts, int64_t D, float c) {
  const int64_t d = blockIdx.x * 128ll + threadIdx.x;
  if (d >= D) return;
  float s = 0.0f;
  for (int64_t p = 0; p < parts; ++p) s += part[p * D + d];
  dlam[d] = -s * c / (1.0f + expf(-lam[d]));
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

// Sizes every kernel here indexes with: batch in a grid's y, token counts in an int (with
// room for a step past the end), 64-bit element offsets.
bool bad_shape(int64_t batch, int64_t seq_len, int64_t dim) {
  return batch < 0 || seq_len < 0 || dim < 0 || batch > 65535 || seq_len > 0x7fff0000LL ||
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
                     final_state, states, static_cast<int>(seq_len), dim, st, static_cast<int>(num_seqs),
                     static_cast<float>(decay_scale), cu_seqlens ? device_error_ptr() : nullptr, Consts()};
  switch (dtype) {
    case TILEOPS_DT_F32: return launch_fwd<float>(args, batch, s);
    case TILEOPS_DT_F16: return launch_fwd<__half>(args, batch, s);
    default: return launch_fwd<__nv_bfloat16>(args, batch, s);
  }
}

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
  const float c = static_cast<float>(decay_scale);
  float* part = static_cast<float*>(workspace);
  const BwdArgs args{dy, x, input_gate, decay_gate, decay_param, states, initial_state,
                     d_final_state, cu_seqlens, dx, d_input_gate, d_decay_gate, part,
                     d_initial_state, static_cast<int>(seq_len), dim, st, static_cast<int>(num_seqs), c,
                     cu_seqlens ? device_error_ptr() : nullptr, Consts()};
  int status;
  switch (dtype) {
    case TILEOPS_DT_F32: status = launch_bwd<float>(args, batch, s); break;
    case TILEOPS_DT_F16: status = launch_bwd<__half>(args, batch, s); break;
    default: status = launch_bwd<__nv_bfloat16>(args, batch, s);
  }
  if (status != TILEOPS_OK) return status;
  const int64_t parts = batch * scan_grid<BwdGeo>(batch, seq_len, dim).cluster;
  glr_dparam<<<static_cast<unsigned>((dim + 127) / 128), 128, 0, s>>>(part, decay_param,
                                                                      d_decay_param, parts, dim, c);
  return launch_status();
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
