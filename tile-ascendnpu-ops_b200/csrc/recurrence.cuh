// Parts shared by the gated linear recurrence's forward and backward kernels: the gates, the
// packed two-channel arithmetic, a warp's tiles, packed sequences, the join of maps
// along the tokens and the launch.
#pragma once

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

// A decay is above zero however strong it is, and so is a product of decays: 2^-149, the least
// float, is added where they could underflow (to no effect on what is 2^-125 or more, on
// NaN and on the mark kForget).  An infinite state so stays infinite, where 0 * inf would
// be NaN; a finite one gains less than 5e-7 at its type's end.  (Half an issue slot an element
// where decays are strong, 1% of the time; a maximum in its place spilled, 10%.)
constexpr float kLeastDecay = 1.401298464324817e-45f;

__device__ __forceinline__ void decay_of(float f, float& a, float& m2) {
  float p = fmaf(f, kG4, kG3);
  p = fmaf(f, p, kG2);
  p = fmaf(f, p, kG1);
  p = fmaf(f, p, kG0);
  const float g = f * p;
  const float e = ex2_approx_f(-kLog2e * f) + kLeastDecay;
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
    const float2 e = fadd2(make_float2(ex2_approx_f(t.x), ex2_approx_f(t.y)), both(kLeastDecay));
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
  Run r(ffma2(first.A, then.A, both(kLeastDecay)), apply<kPacked>(then, first.H));
  if (kPacked) {
    if (first.A.x < 0.0f || then.A.x < 0.0f) r.A.x = kForget;
    if (first.A.y < 0.0f || then.A.y < 0.0f) r.A.y = kForget;
  }
  return r;
}

constexpr int kMaxCluster = 8;  // CTAs of a cluster

// Why this split.  A sequence is a chain, but a run of tokens is a map h -> A h + H that needs
// no predecessor, so runs are worked out side by side, their maps joined, and
// each walked again from its true state: two fma an element more than the
// chain, and every tensor is still read once (DRAM traffic measured within 1% of the
// algorithm's).  Forward, an element takes 32 to 33 issue slots, of which 5 on the
// special-function unit (16 lanes a clock and SM: 37 us of the 41 us that 8 x
// 1024 x 4096 bf16 takes at the copy rate); 16 warps of 128 registers an SM
// keep that unit at 58 to 68% busy (72 us; 8 x 4096 x 4096 215 us, 0.77 of the
// copy rate).  Measured and not taken: 24 warps with runs of 8 tokens, 20%
// slower (twice the joins); a barrier a step in place of the chain of warps,
// 3% slower; 64 channels a CTA, 10% slower (half as many CTAs to fill the SMs).

// How a warp lies over channels and tokens: `Chans` channels side by side, two a lane,
// and groups of lanes one after another in time, `Run` tokens a lane; up to `Warps` warps a
// CTA.  Sixteen warps are what an SM holds of these kernels (128 registers a thread): two
// CTAs of 8, or one of 15 (the links between warps take a hardware barrier
// each, beside that of the CTA).
template <int Chans, int Run, int Warps>
struct Geo {
  static constexpr int kChans = Chans, kRun = Run, kWarps = Warps, kCtas = 16 / Warps;
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
  float4 warp_run[2][G::kWarps][G::kPairs];  // (A, H) of two channels
  float4 cta_run[2][kMaxCluster][G::kPairs];

  // Maps of warps and CTAs that do not exist stay the identity.
  __device__ __forceinline__ void init(int warp, int warps, uint32_t size, int pair) {
    const float4 identity = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
    for (int w = warp; w < G::kWarps; w += warps)
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
      for (int w = 1; w < G::kWarps; ++w)
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
      for (int w = 0; w < G::kWarps - 1; ++w)
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

// ---- launches ----
// The tokens' split over warps and CTAs: a run a warp, up to G::kWarps; then clusters of
// 2, 4 or 8 CTAs along the tokens while twice the CTAs are still resident at once.
struct ScanGrid {
  int warps, cluster;
  int64_t blocks;
};

template <typename G>
ScanGrid scan_grid(int64_t batch, int64_t seq_len, int64_t dim) {
  ScanGrid g;
  g.blocks = (dim + G::kChans - 1) / G::kChans;
  const int64_t runs = (seq_len + G::kWarpRun - 1) / G::kWarpRun;
  g.warps = static_cast<int>(std::min<int64_t>(runs, G::kWarps));
  g.cluster = 1;
  const int64_t resident = static_cast<int64_t>(sm_count()) * G::kCtas;
  while (g.cluster < kMaxCluster && g.blocks * batch * g.cluster * 2 <= resident &&
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

// Sizes every kernel here indexes with: batch in a grid's y, token counts in an int (with
// room for a step past the end), 64-bit element offsets.
inline bool bad_shape(int64_t batch, int64_t seq_len, int64_t dim) {
  return batch < 0 || seq_len < 0 || dim < 0 || batch > 65535 || seq_len > 0x7fff0000LL ||
         dim > 0x7fffffffLL;
}

}  // namespace
}  // namespace tileops
