// Sandwich norm, backward pass.  The formulas and the design are in sandwich_norm.cu.
#include "sandwich_norm.cuh"

namespace tileops {
namespace {

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

template <typename T, typename W, int kThreads, int kPackets, int kStages, int kCtas, int kBytes,
          bool kBias, bool kLayer>
__global__ void __launch_bounds__(kThreads, kCtas) sn_bwd(const BwdArgs p) {
  using C = Cols<T, kThreads, kPackets, kBytes>;
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
      if constexpr (C::kWhole) {
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
          if (!C::kWhole && 2 * i >= n[j]) t[i].x = 0.0f;
          if (!C::kWhole && 2 * i + 1 >= n[j]) t[i].y = 0.0f;
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

// One CTA a stretch of rows: each row's statistics, its outputs, then its share of the
// column sums, which stay in the workspace (a thread adds to its own columns).
template <typename T, typename W, bool kBias, int kV>
__global__ void __launch_bounds__(512) sn_bwd_wide(const BwdArgs p) {
  constexpr int kSums = kBias ? 4 : 2;
  __shared__ float red[32];
  const int64_t N = p.N;
  const int64_t first = static_cast<int64_t>(threadIdx.x) * kV, step = blockDim.x * kV;
  const W *w1 = static_cast<const W*>(p.w1), *w2 = static_cast<const W*>(p.w2);
  const float inv_n = 1.0f / static_cast<float>(N);
  const int64_t row0 = first_row(p.M, blockIdx.x, gridDim.x),
                end = first_row(p.M, blockIdx.x + 1, gridDim.x);
  int64_t group = -1;
  for (int64_t row = row0; row < end; ++row) {
    const int64_t g = row / p.rows_per_group;
    const T *x = static_cast<const T*>(p.x) + row * N, *s = static_cast<const T*>(p.s) + row * N,
            *dy = static_cast<const T*>(p.dy) + row * N,
            *ds = p.ds ? static_cast<const T*>(p.ds) + row * N : nullptr;
    const W* gate = p.gate ? static_cast<const W*>(p.gate) + g * N : nullptr;
    float* to = stretch(p.part, blockIdx.x, g, kSums, p.N);
    const bool fresh = g != group;
    group = g;
    const float2 sx = row_stats<kV>(x, N, p.layer, p.eps, red);
    const float2 ss = row_stats<kV>(s, N, p.layer, p.eps, red);
    float f0 = 0.0f, f1 = 0.0f;
    float sv[kV], gv[kV], w[kV], xv[kV], ga[kV], t[kV];
    for (int64_t c = first; c < N; c += step) {
      load_cols<kV>(s + c, sv);
      load_cols<kV>(dy + c, gv);
      load_vector<kV>(w2, c, 1.0f, p.vec, w);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float f = gv[i] * w[i];
        f0 += f;
        f1 = fmaf(f, (sv[i] - ss.x) * ss.y, f1);
      }
    }
    const float mf = p.layer ? block_sum(f0, red) * inv_n : 0.0f;
    const float mfs = block_sum(f1, red) * inv_n;
    // ds' of a packet (t), with s^ in sv and x^ in xv.
    auto packet = [&](int64_t c) {
      load_cols<kV>(s + c, sv);
      load_cols<kV>(dy + c, gv);
      load_cols<kV>(x + c, xv);
      load_vector<kV>(w2, c, 1.0f, p.vec, w);
      if (ds) {
        load_cols<kV>(ds + c, t);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) t[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        sv[i] = (sv[i] - ss.x) * ss.y;
        xv[i] = (xv[i] - sx.x) * sx.y;
        t[i] = fmaf(ss.y, gv[i] * w[i] - mf - sv[i] * mfs, t[i]);
      }
      load_vector<kV>(w1, c, 1.0f, p.vec, w);
      load_vector<kV>(gate, c, 1.0f, p.vec, ga);
    };
    float e0 = 0.0f, e1 = 0.0f;
    for (int64_t c = first; c < N; c += step) {
      packet(c);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float e = t[i] * ga[i] * w[i];
        e0 += e;
        e1 = fmaf(e, xv[i], e1);
      }
      // This thread's columns of the sums, which it alone adds to.
      auto add = [&](int which, auto term) {
        float a[kV];
        float* at = to + which * N + c;
        if (fresh) {
#pragma unroll
          for (int i = 0; i < kV; ++i) a[i] = 0.0f;
        } else {
          load_cols<kV>(at, a);
        }
#pragma unroll
        for (int i = 0; i < kV; ++i) a[i] += term(i);
        if constexpr (kV % 4 == 0) {
#pragma unroll
          for (int i = 0; i < kV; i += 4)
            *reinterpret_cast<float4*>(at + i) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
        } else {
          at[0] = a[0];
        }
      };
      add(0, [&](int i) { return t[i] * xv[i]; });
      add(1, [&](int i) { return gv[i] * sv[i]; });
      if (kBias) {
        add(2, [&](int i) { return t[i]; });
        add(3, [&](int i) { return gv[i]; });
      }
    }
    const float me = p.layer ? block_sum(e0, red) * inv_n : 0.0f;
    const float mex = block_sum(e1, red) * inv_n;
    for (int64_t c = first; c < N; c += step) {
      packet(c);
      float dr[kV], dx[kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        dr[i] = p.alpha * t[i];
        dx[i] = sx.y * (t[i] * ga[i] * w[i] - me - xv[i] * mex);
      }
      store_cols<kV>(static_cast<T*>(p.dres) + row * N + c, dr);
      store_cols<kV>(static_cast<T*>(p.dx) + row * N + c, dx);
    }
  }
}

// CTAs an SM of the backward pass: for 16-bit rows, as many as their registers allow (each adds
// a stretch of column sums to write and read).  With biases there are twice the sums, and
// a row of 4096 takes more than the 128 registers a thread of two CTAs has (16384 x 4096
// bf16, before the norms were kernels of their own: two CTAs 152 us without and 284 us
// with biases, one 165 and 225 us).  The rule was measured in 16 bits only.  An fp32 row has
// twice the packets and a larger ring: of 513 to 1024 columns, 1025 to 2048 with biases and
// 2049 to 4096 without, half of these CTAs are resident and the others follow them (1025 x
// 1155 LayerNorm with biases 37 us, 0.12 of the copy rate; 8192 x 4096 RMS 147 us, 0.84).
int64_t ctas_per_sm(int64_t N, bool bias) {
  if (N > 8192) return 2;  // the passes over L2, or one CTA at a time of the others
  return N <= 1024 ? 4 : (N <= 2048 ? 2 : (N <= 4096 && !bias ? 2 : 1));
}
constexpr int kMaxSms = 256;  // workspace: more than any device of this architecture has

template <typename T, typename W, int kBytes, bool kBias, bool kLayer>
int launch_bwd(const BwdArgs& a, int64_t ctas, cudaStream_t s) {
  const int64_t packets = (a.N + 16 / sizeof(T) - 1) / (16 / sizeof(T));
  auto go = [&](auto kernel, int threads, int per_thread, int stages) {
    return launch_rows(kernel, threads, static_cast<size_t>(stages) * 4 * per_thread * threads * 16,
                       ctas, a, s);
  };
  if (packets <= 128) return go(sn_bwd<T, W, 128, 1, 6, 4, kBytes, kBias, kLayer>, 128, 1, 6);
  if (packets <= 256) return go(sn_bwd<T, W, 256, 1, 5, 2, kBytes, kBias, kLayer>, 256, 1, 5);
  if (packets <= 512) {
    if constexpr (kBias)
      return go(sn_bwd<T, W, 256, 2, 4, 1, kBytes, kBias, kLayer>, 256, 2, 4);
    else
      return go(sn_bwd<T, W, 256, 2, 3, 2, kBytes, kBias, kLayer>, 256, 2, 3);
  }
  if (packets <= 1024) return go(sn_bwd<T, W, 512, 2, 3, 1, kBytes, kBias, kLayer>, 512, 2, 3);
  sn_bwd_wide<T, W, kBias, kBytes == 16 ? 16 / sizeof(T) : 1>
      <<<static_cast<unsigned>(ctas), 512, 0, s>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace tileops

using namespace tileops;

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
  if (!aligned16(workspace)) return TILEOPS_EALIGN;
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
    const int status = with_bytes<T>(
        N, {dy, d_residual_out, x, residual_out, dx, d_residual}, [&](auto bytes) {
          constexpr int kBytes = decltype(bytes)::value;
          if (bias)
            return args.layer ? launch_bwd<T, W, kBytes, true, true>(args, ctas, st)
                              : launch_bwd<T, W, kBytes, true, false>(args, ctas, st);
          return args.layer ? launch_bwd<T, W, kBytes, false, true>(args, ctas, st)
                            : launch_bwd<T, W, kBytes, false, false>(args, ctas, st);
        });
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
