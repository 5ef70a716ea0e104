// Rotary positions: queries and keys rotated (forward and backward), and new keys and values
// appended to a paged cache with the keys rotated on the way.
//
// Pair i of a head at position p, f_i its angle a token, A an amplitude:
//   c = A cos(p f_i), s = A sin(p f_i);  x'_a = c x_a - s x_b,  x'_b = s x_a + c x_b
// (a, b) = (i, i + R/2) in the half layout, (2i, 2i + 1) in the interleaved one; channels from R
// on pass unchanged.  The backward pass is the transposed map: -s for s.  The arithmetic is fp32,
// rounded once.
//
// Angles.  p f_i in fp32 is off by p f_i 2^-24 radians, 0.06 at a million tokens.  Here f_i is a
// whole number of 2^-64 turns (made on the host in 64 bits): p times it, modulo 2^64, is the
// phase exactly but for p 2^-65 turns, whatever the sign of p.  Its upper 32 bits as a signed
// fraction, less whole quarter turns, go to sincospif: an argument off by 2^-27 half turns at most.
//
// HBM-bound: every channel is read and written once, about 3 flops each.  An item is two vectors of
// a head, 16 bytes each where layouts allow, that hold whole pairs.  A thread keeps one item of a
// token (or of each of several at once, where a token has few items) and walks a tile of tokens with
// it, so that addresses cost two multiplications; the tile's angles are made once, by all threads
// and while the first loads are on their way, and serve all of its heads from shared memory.
// Measured (bf16, in a graph): 8 x 4096 x 64 heads x 128 164 us, the time of a plain copy of as many
// bytes; 8 x 4096 x 40 heads x 128 108 us (0.94); append of 16384 packed tokens x 48 rows x 128 77 us (0.80).
// What did not help: shares of the tokens for as many CTAs as run at once (200 us for the first of
// these), the next token's loads in flight during one's arithmetic (171 us: more registers, fewer CTAs).
#include <algorithm>

#include "common.cuh"
#include "device_error.cuh"

namespace tileops {
namespace {

constexpr int kThreads = 256;  // of a CTA, at most
constexpr int kMaxPairs = 128;  // rotated channels of a head <= 256
constexpr int kTile = 4;        // tokens of a CTA, for each that its threads take at once
constexpr int kMaxTokens = 64;  // of a CTA

// Elements from a batch entry, token and head to the next.
struct RowStrides {
  int64_t b, t, h;
};

struct RotaryArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;  // k_out and v_out: the caches where paged
  RowStrides qs, ks, vs, qo, ko, vo;  // of the caches: page, slot, head
  const void* positions;  // of the tokens, or NULL: 0, 1, ... in each batch entry
  int64_t pos_stride;     // from a batch entry to the next
  int pos64;
  uint32_t tokens;        // in all
  int interleaved;
  int heads, heads_kv, dim, rotary, tile;  // tile: tokens of a CTA
  float amplitude, sign;
  uint32_t per_row, items;  // items of a head, of a token
  uint32_t lanes;           // tokens that a CTA's threads take at once
  uint32_t groups;          // CTAs that share the items of a tile: neighbours, so that they run together
  FastDivU32 div_seq{1}, div_row{1}, div_items{1};  // by the tokens of a batch entry, per_row, items
  // paged
  const int32_t *page_table, *seq_lens, *cu_seqlens;
  int64_t table_stride, num_pages;
  int num_seqs, table_width, page_size;
  int* err;
  uint64_t turns[kMaxPairs];  // 2^64 times the turns a token
};

template <int BYTES>
struct Word;
template <>
struct Word<16> {
  using type = uint4;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<2> {
  using type = uint16_t;
};

template <typename T, int VEC>
union Vec {
  typename Word<VEC * sizeof(T)>::type w;
  T e[VEC];
};

// Loads keep their place before the barrier below and go past L1 (each byte is read once).  They
// are coherent ones: rotated in place, the words read are written later by the same thread.
template <typename T, int VEC>
__device__ __forceinline__ void load(Vec<T, VEC>& v, const T* p) {
  constexpr int kBytes = VEC * sizeof(T);
  if constexpr (kBytes == 16) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.w.x), "=r"(v.w.y), "=r"(v.w.z), "=r"(v.w.w)
                 : "l"(p));
  } else if constexpr (kBytes == 8) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                 : "=r"(v.w.x), "=r"(v.w.y)
                 : "l"(p));
  } else if constexpr (kBytes == 4) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v.w) : "l"(p));
  } else {
    asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];" : "=h"(v.w) : "l"(p));
  }
}

// What a CTA knows of one of its tokens.
struct Token {
  int64_t k_at, v_at;  // its slot in the caches (paged)
  int64_t position;
  int kept;            // bit 0: its queries are rotated (else zeroed), bit 1: it is appended
};

// Sequence of packed token t: the first whose end lies behind t, num_seqs where there is none.  (By
// a warp, 32 ends at a time, the search waits less often, but the call is slower: its registers.)
__device__ __forceinline__ int sequence_of(const int32_t* cu, int num_seqs, int64_t t) {
  int from = 0, to = num_seqs;
  while (from < to) {
    const int middle = (from + to) >> 1;
    if (cu[middle + 1] > t) to = middle; else from = middle + 1;
  }
  return from;
}

__device__ Token appended_token(const RotaryArgs& a, uint32_t token) {
  Token k{0, 0, -1, 0};
  int b;
  if (a.cu_seqlens) {
    b = sequence_of(a.cu_seqlens, a.num_seqs, token);
    if (b == a.num_seqs) return k;  // behind the last sequence
    k.position = a.seq_lens[b] - (a.cu_seqlens[b + 1] - static_cast<int64_t>(token));
  } else {
    b = a.div_seq.div(token);
    k.position = static_cast<int64_t>(a.seq_lens[b]) - a.div_seq.d + (token - b * a.div_seq.d);
  }
  if (k.position < 0) return k;  // padding
  k.kept = 1;
  const int64_t column = k.position / a.page_size;
  const int slot = static_cast<int>(k.position - column * a.page_size);
  if (column < a.table_width) {
    const int64_t page = a.page_table[b * a.table_stride + column];
    if (page >= 0 && page < a.num_pages) {
      k.kept = 3;
      k.k_at = page * a.ko.b + slot * a.ko.t;
      k.v_at = page * a.vo.b + slot * a.vo.t;
    }
  }
  if (k.kept == 1) report_device_error(a.err, kErrBadPage);
  return k;
}

// cos and sin, times the amplitude, of a phase in 2^-32 turns.
__device__ __forceinline__ float2 turn(uint32_t phase, float amplitude) {
  const uint32_t quarters = (phase + 0x20000000u) >> 30;
  const float half_turns = static_cast<int32_t>(phase - (quarters << 30)) * 0x1p-31f;
  float s, c;
  sincospif(half_turns, &s, &c);
  s *= amplitude;
  c *= amplitude;
  const float cq = quarters & 1 ? -s : c, sq = quarters & 1 ? c : s;
  return quarters & 2 ? make_float2(-cq, -sq) : make_float2(cq, sq);
}

// A thread's row: of q, then k, then v.
template <typename T, bool PAGED>
struct Rows {
  const T* src;
  T* dst;
  RowStrides from, to;
  int kind;  // 0 q, 1 k, 2 v
  __device__ __forceinline__ Rows(const RotaryArgs& a, int row) {
    if (row < a.heads) {
      src = static_cast<const T*>(a.q);
      dst = static_cast<T*>(a.q_out);
      from = a.qs;
      to = a.qo;
      kind = 0;
    } else if (!PAGED || row < a.heads + a.heads_kv) {
      row -= a.heads;
      src = static_cast<const T*>(a.k);
      dst = static_cast<T*>(a.k_out);
      from = a.ks;
      to = a.ko;
      kind = 1;
    } else {
      row -= a.heads + a.heads_kv;
      src = static_cast<const T*>(a.v);
      dst = static_cast<T*>(a.v_out);
      from = a.vs;
      to = a.vo;
      kind = 2;
    }
    src += row * from.h;
    dst += row * to.h;
  }
  static __device__ __forceinline__ int64_t place(const RotaryArgs& a, uint32_t token,
                                                  const RowStrides& s) {
    const uint32_t b = a.div_seq.div(token);
    return b * s.b + (token - b * a.div_seq.d) * s.t;
  }
  // Where a token's row goes, or NULL; zeroed: a row of padding.
  __device__ __forceinline__ T* target(const RotaryArgs& a, uint32_t token, const Token& told,
                                       bool& zeroed) const {
    zeroed = false;
    if (PAGED && kind != 0) {
      if (!(told.kept & 2)) return nullptr;
      return dst + (kind == 1 ? told.k_at : told.v_at);
    }
    if (PAGED) zeroed = !(told.kept & 1);
    return dst + place(a, token, to);
  }
};

// cu_seqlens as a whole, by one CTA.
__device__ __forceinline__ void check_offsets(const RotaryArgs& a) {
  bool bad = threadIdx.x == 0 && (a.cu_seqlens[0] != 0 ||
                                  a.cu_seqlens[a.num_seqs] > static_cast<int64_t>(a.tokens));
  for (int n = threadIdx.x; n < a.num_seqs; n += blockDim.x)
    bad |= a.cu_seqlens[n] > a.cu_seqlens[n + 1];
  if (bad) report_device_error(a.err, kErrBadSeqlens);
}

// cos and (signed) sin of every pair of a tile's tokens, by the whole CTA, to put(token, pair, cos, sin).
template <bool PAGED, typename Put>
__device__ __forceinline__ void make_angles(const RotaryArgs& a, uint32_t token0, int ntok,
                                            Token* told, Put put) {
  if (PAGED) {
    if (threadIdx.x < ntok) told[threadIdx.x] = appended_token(a, token0 + threadIdx.x);
    if (a.cu_seqlens && blockIdx.x == 0) check_offsets(a);
    __syncthreads();
  }
  const int pairs = a.rotary / 2;
  for (int n = threadIdx.x; n < ntok * pairs; n += blockDim.x) {
    const int at = n / pairs, i = n - at * pairs;
    int64_t position;
    if (PAGED) {
      position = told[at].position;
    } else {
      const uint32_t b = a.div_seq.div(token0 + at), t = token0 + at - b * a.div_seq.d;
      const int64_t place = b * a.pos_stride + t;
      position = !a.positions ? t
                 : a.pos64    ? static_cast<const int64_t*>(a.positions)[place]
                              : static_cast<const int32_t*>(a.positions)[place];
    }
    const float2 w = turn(static_cast<uint32_t>((static_cast<uint64_t>(position) * a.turns[i]) >> 32),
                          a.amplitude);
    put(at, i, w.x, a.sign * w.y);
  }
}

template <typename T, int VEC, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kThreads, 5) rotary_rows(const __grid_constant__ RotaryArgs a) {
  __shared__ Token told[PAGED ? kMaxTokens : 1];
  // [token], then as the items read them (16 bytes and no bank twice in 8 threads): two pairs' cos and
  // sin together, those of the items' first pairs, of their next, ...
  extern __shared__ __align__(16) float angles[];
  constexpr int kTwo = VEC % 2 == 0 ? 2 : 1;  // pairs together
  const uint32_t column = blockIdx.x / a.groups, group = blockIdx.x - column * a.groups;
  const uint32_t token0 = column * static_cast<uint32_t>(a.tile);
  const int ntok = min(static_cast<uint32_t>(a.tile), a.tokens - token0);
  const int pairs = a.rotary / 2;

  // ---- this thread's item ----
  const int lane = a.lanes == 1 ? 0 : a.div_items.div(threadIdx.x);
  const uint32_t item = group * blockDim.x + threadIdx.x - lane * a.items;
  const bool mine = item < a.items && lane < a.lanes;
  const uint32_t row = a.div_row.div(item), j = item - row * a.per_row;
  const bool in_turn = j < static_cast<uint32_t>(pairs / VEC);
  const int pair = j * VEC;  // the first of its pairs
  int ca, cb;                // its channels; cb < 0: no second vector
  if (in_turn) {
    ca = INTER ? 2 * pair : pair;
    cb = ca + (INTER ? VEC : pairs);
  } else {
    ca = a.rotary + (j - pairs / VEC) * 2 * VEC;
    cb = ca + VEC < a.dim ? ca + VEC : -1;
  }
  const Rows<T, PAGED> rows(a, row);
  const bool turns = in_turn && rows.kind != 2;

  Vec<T, VEC> x, y;
  auto fetch = [&](int at) {
    if (!mine || at >= ntok) return;
    const T* p = rows.src + rows.place(a, token0 + at, rows.from);
    load<T, VEC>(x, p + ca);
    if (cb >= 0) load<T, VEC>(y, p + cb);
  };
  fetch(lane);

  // ---- the tile's angles ----
  make_angles<PAGED>(a, token0, ntok, told, [&](int at, int i, float c, float sn) {
    const int of = i / VEC, r = i - of * VEC;
    float* const to = angles + at * a.rotary + ((r / kTwo) * (pairs / VEC) + of) * 2 * kTwo + r % kTwo;
    to[0] = c;
    to[kTwo] = sn;
  });
  __syncthreads();

  for (int at = lane; at < ntok; at += a.lanes) {
    if (!mine) break;
    if (at != lane) fetch(at);
    if (turns) {
      const float* w = angles + at * a.rotary + j * 2 * kTwo;
      if constexpr (VEC % 2 == 0) {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float4 cs = *reinterpret_cast<const float4*>(w + e * (pairs / VEC) * 2);
          const float2 c2 = make_float2(cs.x, cs.y), s2 = make_float2(cs.z, cs.w);
          T* const first = INTER ? (2 * e < VEC ? x.e + 2 * e : y.e + (2 * e - VEC)) : x.e + e;
          T* const other = !INTER             ? y.e + e
                           : 2 * e + 2 < VEC ? x.e + 2 * e + 2
                                             : y.e + (2 * e + 2 - VEC);
          // INTER: pairs (0, 1) of `first` and `other` each; else pairs across the two vectors.
          const float2 a2 = INTER ? make_float2(Cvt<T>::to_f(first[0]), Cvt<T>::to_f(other[0]))
                                  : make_float2(Cvt<T>::to_f(first[0]), Cvt<T>::to_f(first[1]));
          const float2 b2 = INTER ? make_float2(Cvt<T>::to_f(first[1]), Cvt<T>::to_f(other[1]))
                                  : make_float2(Cvt<T>::to_f(other[0]), Cvt<T>::to_f(other[1]));
          const float2 sb = fmul2(s2, b2);
          const float2 ra = ffma2(c2, a2, make_float2(-sb.x, -sb.y));
          const float2 rb = ffma2(c2, b2, fmul2(s2, a2));
          first[0] = Cvt<T>::from_f(ra.x);
          (INTER ? other[0] : first[1]) = Cvt<T>::from_f(ra.y);
          (INTER ? first[1] : other[0]) = Cvt<T>::from_f(rb.x);
          other[1] = Cvt<T>::from_f(rb.y);
        }
      } else {
        const float xa = Cvt<T>::to_f(x.e[0]), xb = Cvt<T>::to_f(y.e[0]);
        x.e[0] = Cvt<T>::from_f(fmaf(w[0], xa, -(w[1] * xb)));
        y.e[0] = Cvt<T>::from_f(fmaf(w[0], xb, w[1] * xa));
      }
    }
    bool zeroed;
    T* const p = rows.target(a, token0 + at, told[PAGED ? at : 0], zeroed);
    if (!p) continue;
    if (zeroed) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x.e[e] = y.e[e] = Cvt<T>::from_f(0.0f);
    }
    *reinterpret_cast<decltype(x.w)*>(p + ca) = x.w;
    if (cb >= 0) *reinterpret_cast<decltype(y.w)*>(p + cb) = y.w;
  }
}

// Where the two channels of a pair do not lie whole vectors apart (half of the rotated channels is odd,
// say), a vector of channels is loaded as it lies and its partners come through shared memory (interleaved:
// they are in the vector): a thread keeps one vector of one row over the tile's tokens, angles are laid out
// by channel with the sine's sign in place.  Words a quarter as wide in the form above take longer (6123
// tokens x 48 rows x 128 bf16, 30 channels rotated, 94 us and 45), words half as wide do not (19488 x 20 x
// 96, 8 rotated, 35 and 47).  A copy would take 23 us for either: here the threads meet at a barrier for
// each group of tokens, there the channels that pass move in the pairs' narrow words too.
template <typename T, int VEC, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kThreads, 4) rotary_staged(const __grid_constant__ RotaryArgs a) {
  __shared__ Token told[PAGED ? kMaxTokens : 1];
  __shared__ __align__(16) Vec<T, VEC> stage[INTER ? 1 : 2][INTER ? 1 : kThreads];
  extern __shared__ __align__(16) float angles[];  // [token][cos, sin][channel]
  const uint32_t column = blockIdx.x / a.groups, group = blockIdx.x - column * a.groups;
  const uint32_t token0 = column * static_cast<uint32_t>(a.tile);
  const int ntok = min(static_cast<uint32_t>(a.tile), a.tokens - token0);
  const int wide = (a.rotary + VEC - 1) / VEC * VEC;  // channels of an angle table

  // ---- this thread's vector: of row `row` of the group's, of token `lane` of those at once ----
  const int lane = a.lanes == 1 ? 0 : a.div_items.div(threadIdx.x);
  const uint32_t item = threadIdx.x - lane * a.items;  // items: of a group here
  const uint32_t row = a.div_row.div(item), j = item - row * a.per_row;
  const uint32_t row_all = group * (a.items / a.per_row) + row;
  const bool mine = item < a.items && lane < a.lanes &&
                    row_all < static_cast<uint32_t>(a.heads + (PAGED ? 2 : 1) * a.heads_kv);
  const int channel = j * VEC;
  const Rows<T, PAGED> rows(a, mine ? row_all : 0);
  const bool turns = mine && rows.kind != 2 && channel < a.rotary;

  Vec<T, VEC> x;
  auto fetch = [&](int at) {
    if (mine && at < ntok)
      load<T, VEC>(x, rows.src + rows.place(a, token0 + at, rows.from) + channel);
  };
  fetch(lane);
  make_angles<PAGED>(a, token0, ntok, told, [&](int at, int i, float c, float sn) {
    const int first = INTER ? 2 * i : i, other = INTER ? first + 1 : i + a.rotary / 2;
    float* const to = angles + at * 2 * wide;
    to[first] = to[other] = c;
    to[wide + first] = -sn;
    to[wide + other] = sn;
  });
  int buf = 0;
  for (int begin = 0; begin < ntok; begin += a.lanes, buf ^= 1) {
    const int at = begin + lane;
    Vec<T, VEC> v = x;
    if (!INTER) stage[buf][threadIdx.x] = v;
    fetch(at + a.lanes);
    if (!INTER || begin == 0) __syncthreads();  // also of the angles, the first time
    if (!mine || at >= ntok) continue;
    if (turns) {
      const float* const w = angles + at * 2 * wide + channel;
      const T* const head = reinterpret_cast<const T*>(stage[INTER ? 0 : buf]) + (threadIdx.x - j) * VEC;
      const int half = a.rotary / 2;
      const Vec<T, VEC> own = v;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int d = channel + e;
        if (d >= a.rotary) continue;
        const float p = Cvt<T>::to_f(INTER ? own.e[e ^ 1] : head[d < half ? d + half : d - half]);
        v.e[e] = Cvt<T>::from_f(fmaf(w[e], Cvt<T>::to_f(v.e[e]), w[wide + e] * p));
      }
    }
    bool zeroed;
    T* const p = rows.target(a, token0 + at, told[PAGED ? at : 0], zeroed);
    if (!p) continue;
    if (zeroed) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v.e[e] = Cvt<T>::from_f(0.0f);
    }
    *reinterpret_cast<decltype(v.w)*>(p + channel) = v.w;
  }
}

// Whether rows at p with these strides can be read and written in words of `vec` elements.
bool fits(const void* p, const RowStrides& s, int vec, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % (vec * size) == 0 && s.b % vec == 0 && s.t % vec == 0 &&
         s.h % vec == 0;
}

// Tile, CTAs and launch of either kernel; `items` of a token in `groups` CTAs side by side, `room` floats of
// angles a token.
template <typename K>
int launch_tiles(RotaryArgs& a, K kernel, uint32_t items, uint32_t groups, uint32_t threads, int room,
                 cudaStream_t s) {
  // kTile tokens for each that is taken at once, while that makes four CTAs an SM.  (Tiles of 8 and 16
  // were slower, 8 x 4096 x 64 heads x 128 bf16 174 and 188 us for 165: CTAs that run together then
  // lie further apart in memory.)
  const int64_t spread = static_cast<int64_t>(a.tokens) * groups / (4 * sm_count() * a.lanes);
  a.tile = static_cast<int>(a.lanes * std::min<int64_t>(kTile, std::max<int64_t>(spread, 1)));
  a.items = items;
  a.groups = groups;
  a.div_row = FastDivU32(a.per_row);
  a.div_items = FastDivU32(items);
  const int64_t grid = static_cast<int64_t>((a.tokens + a.tile - 1) / a.tile) * groups;
  if (grid > 0x7fffffffLL) return TILEOPS_EBADSHAPE;
  // At least a thread for each token of the tile.
  threads = (std::max(threads, static_cast<uint32_t>(a.tile)) + 31) / 32 * 32;
  const size_t smem = static_cast<size_t>(a.tile) * room * sizeof(float);
  kernel<<<static_cast<unsigned>(grid), threads, smem, s>>>(a);
  return launch_status();
}

// Tokens side by side: as their items fit a CTA, and their tile's angles 16 KB.
uint32_t lanes_of(uint32_t items, int room) {
  const uint32_t fit = std::min(kMaxTokens / kTile, 1024 / std::max(room, 1));
  return std::max<uint32_t>(1, std::min<uint32_t>(kThreads / items, fit));
}

template <typename T, int VEC, bool PAGED>
int launch_vec(RotaryArgs& a, cudaStream_t s) {
  a.per_row = a.rotary / (2 * VEC) + (a.dim - a.rotary + 2 * VEC - 1) / (2 * VEC);
  const uint32_t items = (a.heads + (PAGED ? 2 : 1) * a.heads_kv) * a.per_row;
  // The items of a token in as many CTAs as they need, in equal parts of whole warps.
  const uint32_t groups = (items + kThreads - 1) / kThreads;
  a.lanes = lanes_of(items, a.rotary);
  const uint32_t threads = ((items + groups - 1) / groups * a.lanes + 31) / 32 * 32;
  return launch_tiles(
      a, a.interleaved ? rotary_rows<T, VEC, true, PAGED> : rotary_rows<T, VEC, false, PAGED>, items,
      groups, threads, a.rotary, s);
}

template <typename T, int VEC, bool PAGED>
int launch_staged(RotaryArgs& a, cudaStream_t s) {
  a.per_row = a.dim / VEC;  // at most kThreads
  const uint32_t rows = a.heads + (PAGED ? 2 : 1) * a.heads_kv;
  // Whole rows in a CTA, in equal parts.
  const uint32_t most = kThreads / a.per_row, groups = (rows + most - 1) / most;
  const uint32_t items = (rows + groups - 1) / groups * a.per_row;
  const int room = 2 * ((a.rotary + VEC - 1) / VEC * VEC);
  a.lanes = groups == 1 ? lanes_of(items, room) : 1;
  return launch_tiles(
      a, a.interleaved ? rotary_staged<T, VEC, true, PAGED> : rotary_staged<T, VEC, false, PAGED>, items,
      groups, items * a.lanes, room, s);
}

template <typename T, bool PAGED>
int launch_type(RotaryArgs& a, cudaStream_t s) {
  const int pairs = a.rotary / 2;
  auto rows_fit = [&](int vec) {  // rows in words of vec elements
    bool ok = a.dim % vec == 0;
    if (a.heads) ok = ok && fits(a.q, a.qs, vec, sizeof(T)) && fits(a.q_out, a.qo, vec, sizeof(T));
    if (a.heads_kv)
      ok = ok && fits(a.k, a.ks, vec, sizeof(T)) && fits(a.k_out, a.ko, vec, sizeof(T));
    if (PAGED) ok = ok && fits(a.v, a.vs, vec, sizeof(T)) && fits(a.v_out, a.vo, vec, sizeof(T));
    return ok;
  };
  constexpr int kFull = 16 / sizeof(T);
  int wide = kFull;
  while (wide > 1 && !rows_fit(wide)) wide /= 2;
  int narrow = wide;  // and pairs whole words apart
  while (narrow > 1 && (pairs % narrow != 0 || (a.dim - a.rotary) % narrow != 0)) narrow /= 2;
  if (4 * narrow <= wide && a.dim / wide <= kThreads) {
    if (wide == kFull) return launch_staged<T, kFull, PAGED>(a, s);
    return launch_staged<T, 4, PAGED>(a, s);
  }
  if (narrow == kFull) return launch_vec<T, kFull, PAGED>(a, s);
  if (narrow == kFull / 2) return launch_vec<T, kFull / 2, PAGED>(a, s);
  if constexpr (kFull > 4) {
    if (narrow == 2) return launch_vec<T, 2, PAGED>(a, s);
  }
  return launch_vec<T, 1, PAGED>(a, s);
}

template <bool PAGED>
int launch(RotaryArgs& a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case TILEOPS_DT_F32: return launch_type<float, PAGED>(a, s);
    case TILEOPS_DT_F16: return launch_type<__half, PAGED>(a, s);
    default: return launch_type<__nv_bfloat16, PAGED>(a, s);
  }
}

bool bad_heads(int64_t heads, int64_t heads_kv, int64_t dim, int64_t rotary) {
  return heads < 0 || heads_kv < 0 || heads > 4096 || heads_kv > 4096 || dim < 1 || dim > 4096 ||
         rotary < 0 || rotary > dim || rotary > 2 * kMaxPairs || rotary % 2 != 0;
}

RowStrides strides(const int64_t* s) { return {s[0], s[1], s[2]}; }

}  // namespace
}  // namespace tileops

using namespace tileops;

extern "C" int tileops_rotary(const void* q, const void* k, const void* positions, void* q_out,
                              void* k_out, const uint64_t* turns, int64_t batch, int64_t seq_len,
                              int64_t heads, int64_t heads_kv, int64_t dim, int64_t rotary_dim,
                              const int64_t* strides12, int64_t position_stride,
                              int position_dtype, int interleaved, int backward, double amplitude,
                              int dtype, void* stream) {
  if (batch < 0 || seq_len < 0 || batch > 0x7fffffffLL || seq_len > 0x7fffffffLL ||
      batch * seq_len > 0x7fffffffLL ||
      bad_heads(heads, heads_kv, dim, rotary_dim))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (batch == 0 || seq_len == 0 || heads + heads_kv == 0) return TILEOPS_OK;
  if ((heads && (!q || !q_out)) || (heads_kv && (!k || !k_out)) || !strides12 ||
      (rotary_dim && !turns))
    return TILEOPS_EINVAL;
  if (positions && position_dtype != TILEOPS_DT_I32 && position_dtype != TILEOPS_DT_I64)
    return TILEOPS_EBADDTYPE;
  RotaryArgs a{};
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  a.qs = strides(strides12);
  a.ks = strides(strides12 + 3);
  a.qo = strides(strides12 + 6);
  a.ko = strides(strides12 + 9);
  a.positions = positions;
  a.pos_stride = position_stride;
  a.pos64 = position_dtype == TILEOPS_DT_I64;
  a.div_seq = FastDivU32(static_cast<uint32_t>(seq_len));
  a.tokens = static_cast<uint32_t>(batch * seq_len);
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.dim = static_cast<int>(dim);
  a.rotary = static_cast<int>(rotary_dim);
  a.amplitude = static_cast<float>(amplitude);
  a.sign = backward ? -1.0f : 1.0f;
  std::copy_n(turns, rotary_dim / 2, a.turns);
  a.interleaved = interleaved != 0;
  return launch<false>(a, dtype, as_stream(stream));
}

extern "C" int tileops_paged_kv_append(
    const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,
    const int32_t* page_table, const int32_t* seq_lens, const int32_t* cu_seqlens,
    const uint64_t* turns, int64_t num_seqs, int64_t tokens, int64_t heads, int64_t heads_kv,
    int64_t dim, int64_t rotary_dim, int64_t num_pages, int64_t page_size, int64_t table_width,
    int64_t table_stride, const int64_t* strides18, int interleaved, double amplitude, int dtype,
    void* stream) {
  if (num_seqs < 0 || tokens < 0 || num_seqs > 0x3fffffffLL || tokens > 0x7fffffffLL ||
      num_pages < 0 || num_pages > 0x7fffffffLL || page_size < 1 || page_size > 0x7fffffffLL ||
      table_width < 0 || table_width > 0x7fffffffLL || heads_kv < 1 ||
      bad_heads(heads, heads_kv, dim, rotary_dim) ||
      (!cu_seqlens && (num_seqs ? tokens % num_seqs : tokens) != 0))
    return TILEOPS_EBADSHAPE;
  if (!is_float_dtype(dtype)) return TILEOPS_EBADDTYPE;
  if (tokens == 0) return TILEOPS_OK;
  if ((heads && (!q || !q_out)) || !k || !v || !k_cache || !v_cache || k_cache == v_cache ||
      !strides18 || (num_seqs && !seq_lens) || (num_seqs && table_width && !page_table) ||
      (rotary_dim && !turns))
    return TILEOPS_EINVAL;
  RotaryArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.k_out = k_cache;
  a.v_out = v_cache;
  a.qs = strides(strides18);
  a.ks = strides(strides18 + 3);
  a.vs = strides(strides18 + 6);
  a.qo = strides(strides18 + 9);
  a.ko = strides(strides18 + 12);
  a.vo = strides(strides18 + 15);
  // Packed: one batch entry of all tokens.
  a.div_seq = FastDivU32(static_cast<uint32_t>(cu_seqlens ? tokens : tokens / num_seqs));
  a.tokens = static_cast<uint32_t>(tokens);
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.dim = static_cast<int>(dim);
  a.rotary = static_cast<int>(rotary_dim);
  a.amplitude = static_cast<float>(amplitude);
  a.sign = 1.0f;
  a.page_table = page_table;
  a.seq_lens = seq_lens;
  a.cu_seqlens = cu_seqlens;
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.num_seqs = static_cast<int>(num_seqs);
  a.table_width = static_cast<int>(table_width);
  a.page_size = static_cast<int>(page_size);
  a.err = device_error_ptr();
  std::copy_n(turns, rotary_dim / 2, a.turns);
  a.interleaved = interleaved != 0;
  return launch<true>(a, dtype, as_stream(stream));
}
