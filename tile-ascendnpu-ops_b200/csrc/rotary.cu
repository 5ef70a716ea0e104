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
// fraction go to sincospif: an argument off by 2^-25 half turns at most.
// The angles of a token are made once by its CTA and serve all of its heads.
//
// HBM-bound: every channel is read and written once, about 3 flops each.
#include <algorithm>

#include "common.cuh"
#include "device_error.cuh"

namespace tileops {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // rotated channels of a head <= 256
constexpr int kMaxTokens = 16;  // of a CTA

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
  int seq_len;            // tokens of a batch entry
  int64_t tokens;         // in all
  int heads, heads_kv, dim, rotary, tokens_cta;
  float amplitude, sign;
  uint32_t per_row;       // items of a head: pairs of vectors
  FastDivU32 div_token{1}, div_row{1};
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

// Sequence of packed token t: the first whose end lies behind t, num_seqs where there is none.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int num_seqs, int64_t t) {
  int lo = 0, hi = num_seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__device__ Token appended_token(const RotaryArgs& a, int64_t token) {
  Token k{0, 0, -1, 0};
  int b;
  if (a.cu_seqlens) {
    b = sequence_of(a.cu_seqlens, a.num_seqs, token);
    if (b == a.num_seqs) return k;  // behind the last sequence
    k.position = a.seq_lens[b] - (a.cu_seqlens[b + 1] - token);
  } else {
    b = static_cast<int>(token / a.seq_len);
    k.position = static_cast<int64_t>(a.seq_lens[b]) - a.seq_len + token % a.seq_len;
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

// One CTA: tokens_cta tokens, all heads.  An item is two vectors of VEC channels of a head that
// hold VEC pairs (or up to 2 VEC channels behind the rotated ones); a thread keeps kBatch items'
// loads in flight, the first of them while the angles are made.
template <typename T, int VEC, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kThreads) rotary_rows(const __grid_constant__ RotaryArgs a) {
  constexpr int kBatch = 4;
  __shared__ Token told[kMaxTokens];
  extern __shared__ float2 angles[];  // [token][pair]
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.tokens_cta;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(a.tokens_cta), a.tokens - token0));
  const int pairs = a.rotary / 2;
  const uint32_t rows = a.heads + (PAGED ? 2 : 1) * a.heads_kv;
  const uint32_t items = ntok * rows * a.per_row;
  const uint32_t turned = pairs / VEC;  // items of a head that rotate

  struct Item {
    Vec<T, VEC> x, y;
    int token, row, ca, cb;  // row: of q, then k, then v; ca < 0: no item; cb < 0: no second vector
    int pair;                // < 0: passes unchanged
  };
  Item it[kBatch];

  auto fetch = [&](uint32_t base) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      Item& m = it[u];
      const uint32_t at = base + u * kThreads;
      m.ca = -1;
      if (at >= items) continue;
      m.token = a.div_token.div(at);
      const uint32_t rest = at - m.token * (rows * a.per_row);
      m.row = a.div_row.div(rest);
      const uint32_t j = rest - m.row * a.per_row;
      if (j < turned) {
        m.pair = j * VEC;
        m.ca = INTER ? 2 * j * VEC : j * VEC;
        m.cb = m.ca + (INTER ? VEC : pairs);
      } else {
        m.pair = -1;
        m.ca = a.rotary + (j - turned) * 2 * VEC;
        m.cb = m.ca + VEC < a.dim ? m.ca + VEC : -1;
      }
      const int64_t token = token0 + m.token;
      int64_t b = 0, t = token;
      if (!PAGED || !a.cu_seqlens) {
        b = token / a.seq_len;
        t = token - b * a.seq_len;
      }
      int h = m.row;
      const void* src = a.q;
      const RowStrides* s = &a.qs;
      if (h >= a.heads) {
        h -= a.heads;
        src = a.k;
        s = &a.ks;
        if (PAGED && h >= a.heads_kv) {
          h -= a.heads_kv;
          src = a.v;
          s = &a.vs;
          m.pair = -1;
        }
      }
      const T* p = static_cast<const T*>(src) + b * s->b + t * s->t + h * s->h;
      load<T, VEC>(m.x, p + m.ca);
      if (m.cb >= 0) load<T, VEC>(m.y, p + m.cb);
    }
  };

  fetch(threadIdx.x);

  if (PAGED) {
    if (threadIdx.x < ntok) told[threadIdx.x] = appended_token(a, token0 + threadIdx.x);
    if (a.cu_seqlens && blockIdx.x == 0) {
      bool bad = threadIdx.x == 0 && (a.cu_seqlens[0] != 0 || a.cu_seqlens[a.num_seqs] > a.tokens);
      for (int n = threadIdx.x; n < a.num_seqs; n += kThreads)
        bad |= a.cu_seqlens[n] > a.cu_seqlens[n + 1];
      if (bad) report_device_error(a.err, kErrBadSeqlens);
    }
    __syncthreads();
  }
  for (int n = threadIdx.x; n < ntok * pairs; n += kThreads) {
    const int token = n / pairs, i = n - token * pairs;
    int64_t position;
    if (PAGED) {
      position = told[token].position;
    } else {
      const int64_t b = (token0 + token) / a.seq_len, t = token0 + token - b * a.seq_len;
      const int64_t at = b * a.pos_stride + t;
      position = !a.positions ? t
                 : a.pos64    ? static_cast<const int64_t*>(a.positions)[at]
                              : static_cast<const int32_t*>(a.positions)[at];
    }
    const uint64_t phase = static_cast<uint64_t>(position) * a.turns[i];
    const float half_turns = static_cast<int32_t>(phase >> 32) * 0x1p-31f;
    float s, c;
    sincospif(half_turns, &s, &c);
    angles[n] = make_float2(a.amplitude * c, a.sign * a.amplitude * s);
  }
  __syncthreads();

  for (uint32_t base = threadIdx.x; base < items; base += kBatch * kThreads) {
    if (base != threadIdx.x) fetch(base);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      Item& m = it[u];
      if (m.ca < 0) continue;
      if (m.pair >= 0) {
        const float2* w = angles + m.token * pairs + m.pair;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          T& first = INTER ? (2 * e < VEC ? m.x.e[2 * e % VEC] : m.y.e[2 * e - VEC]) : m.x.e[e];
          T& second = INTER ? (2 * e + 1 < VEC ? m.x.e[(2 * e + 1) % VEC] : m.y.e[2 * e + 1 - VEC])
                            : m.y.e[e];
          const float c = w[e].x, s = w[e].y;
          const float xa = Cvt<T>::to_f(first), xb = Cvt<T>::to_f(second);
          first = Cvt<T>::from_f(c * xa - s * xb);
          second = Cvt<T>::from_f(s * xa + c * xb);
        }
      }
      const int64_t token = token0 + m.token;
      int64_t b = 0, t = token;
      if (!PAGED || !a.cu_seqlens) {
        b = token / a.seq_len;
        t = token - b * a.seq_len;
      }
      T* p;
      if (m.row < a.heads) {
        p = static_cast<T*>(a.q_out) + b * a.qo.b + t * a.qo.t + m.row * a.qo.h;
        if (PAGED && !(told[m.token].kept & 1)) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) m.x.e[e] = m.y.e[e] = Cvt<T>::from_f(0.0f);
        }
      } else if (!PAGED) {
        p = static_cast<T*>(a.k_out) + b * a.ko.b + t * a.ko.t + (m.row - a.heads) * a.ko.h;
      } else {
        if (!(told[m.token].kept & 2)) continue;
        const int h = m.row - a.heads;
        p = h < a.heads_kv ? static_cast<T*>(a.k_out) + told[m.token].k_at + h * a.ko.h
                           : static_cast<T*>(a.v_out) + told[m.token].v_at +
                                 (h - a.heads_kv) * a.vo.h;
      }
      *reinterpret_cast<decltype(m.x.w)*>(p + m.ca) = m.x.w;
      if (m.cb >= 0) *reinterpret_cast<decltype(m.y.w)*>(p + m.cb) = m.y.w;
    }
  }
}

// Whether rows at p with these strides can be read and written in words of `vec` elements.
bool fits(const void* p, const RowStrides& s, int vec, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % (vec * size) == 0 && s.b % vec == 0 && s.t % vec == 0 &&
         s.h % vec == 0;
}

template <typename T, int VEC, bool PAGED>
int launch_vec(RotaryArgs& a, bool interleaved, cudaStream_t s) {
  a.per_row = a.rotary / (2 * VEC) + (a.dim - a.rotary + 2 * VEC - 1) / (2 * VEC);
  const uint32_t rows = a.heads + (PAGED ? 2 : 1) * a.heads_kv;
  const uint32_t per_token = rows * a.per_row;
  a.div_token = FastDivU32(per_token);
  a.div_row = FastDivU32(a.per_row);
  // Enough tokens a CTA for one batch of loads a thread, as long as every SM has some.
  const int64_t full = std::max<int64_t>(1, 4 * kThreads / per_token);
  const int64_t spread = std::max<int64_t>(1, a.tokens / (2 * sm_count()));
  a.tokens_cta = static_cast<int>(std::min<int64_t>({full, spread, kMaxTokens}));
  const int64_t grid = (a.tokens + a.tokens_cta - 1) / a.tokens_cta;
  if (grid > 0x7fffffffLL) return TILEOPS_EBADSHAPE;
  const size_t smem = static_cast<size_t>(a.tokens_cta) * (a.rotary / 2) * sizeof(float2);
  auto kernel = interleaved ? rotary_rows<T, VEC, true, PAGED> : rotary_rows<T, VEC, false, PAGED>;
  kernel<<<static_cast<unsigned>(grid), kThreads, smem, s>>>(a);
  return launch_status();
}

template <typename T, bool PAGED>
int launch_type(RotaryArgs& a, bool interleaved, cudaStream_t s) {
  auto vector = [&](int vec) {
    const int pairs = a.rotary / 2;
    bool ok = pairs % vec == 0 && (a.dim - a.rotary) % vec == 0 && a.dim % vec == 0;
    if (a.heads) ok = ok && fits(a.q, a.qs, vec, sizeof(T)) && fits(a.q_out, a.qo, vec, sizeof(T));
    if (a.heads_kv)
      ok = ok && fits(a.k, a.ks, vec, sizeof(T)) && fits(a.k_out, a.ko, vec, sizeof(T));
    if (PAGED) ok = ok && fits(a.v, a.vs, vec, sizeof(T)) && fits(a.v_out, a.vo, vec, sizeof(T));
    return ok;
  };
  constexpr int kFull = 16 / sizeof(T);
  if (vector(kFull)) return launch_vec<T, kFull, PAGED>(a, interleaved, s);
  if (vector(kFull / 2)) return launch_vec<T, kFull / 2, PAGED>(a, interleaved, s);
  if constexpr (kFull > 4) {
    if (vector(2)) return launch_vec<T, 2, PAGED>(a, interleaved, s);
  }
  return launch_vec<T, 1, PAGED>(a, interleaved, s);
}

template <bool PAGED>
int launch(RotaryArgs& a, bool interleaved, int dtype, cudaStream_t s) {
  switch (dtype) {
    case TILEOPS_DT_F32: return launch_type<float, PAGED>(a, interleaved, s);
    case TILEOPS_DT_F16: return launch_type<__half, PAGED>(a, interleaved, s);
    default: return launch_type<__nv_bfloat16, PAGED>(a, interleaved, s);
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
  a.seq_len = static_cast<int>(seq_len);
  a.tokens = batch * seq_len;
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.dim = static_cast<int>(dim);
  a.rotary = static_cast<int>(rotary_dim);
  a.amplitude = static_cast<float>(amplitude);
  a.sign = backward ? -1.0f : 1.0f;
  std::copy_n(turns, rotary_dim / 2, a.turns);
  return launch<false>(a, interleaved != 0, dtype, as_stream(stream));
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
  if ((heads && (!q || !q_out)) || !k || !v || !k_cache || !v_cache ||
      !strides18 || (num_seqs && !seq_lens) || (num_seqs && table_width && !page_table) || (rotary_dim && !turns))
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
  a.seq_len = static_cast<int>(cu_seqlens ? tokens : tokens / num_seqs);
  a.tokens = tokens;
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
  return launch<true>(a, interleaved != 0, dtype, as_stream(stream));
}
