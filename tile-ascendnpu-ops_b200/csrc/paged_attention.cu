// Attention of one new token of every sequence over a paged cache of keys and values.
//
//   o   = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j)      (per sequence b, query head h)
//   lse = log2(sum_j w_j)
//
// over the tokens max(0, len_b - window) <= j < len_b; token j lies in slot j % P of page
// page_table[b][j / P].  q (B, H, D); the caches (pages, P, Hkv, D) with any strides that are
// multiples of 16 bytes; query head h reads key head h / (H / Hkv).  A sequence without a token
// has o = 0 and lse = -inf.
//
// Every key and value is read once, 2 D e bytes for 4 D (H / Hkv) flops a token and key head: H / Hkv
// flops a byte, 1 to 16 as a rule, so HBM bounds it.  8 flops a byte at the memory's rate are 52
// TFLOP/s, which the fp32 pipes do not reach beside the conversions; the two products go to the tensor
// cores as m16n8k16 (the query heads of a key head are the 16 rows, or 8 of them; a 128-row tcgen05 tile
// would be 7/8 padding and would take the scores through TMEM and back, for rates not needed here).
//
// The split.  The tokens of each (sequence, key head) are cut into units of 16 or 32 for each warp of
// a CTA, and all units of the call in a row are shared out evenly, a run of them to each CTA,
// whatever the sequences' lengths are (they stay on the device).  An item (sequence and key head)
// whose units lie in one CTA is finished there; of one that lies in several, each writes its sums
// and counts itself, and the last one to do so joins them all, in the order of the CTAs, so that
// results repeat to the bit.  A CTA has at most two items it shares with others: its first and its
// last.  (A second kernel for the joins cost 5 to 7 us a call.)  The counters are zero at the start
// and whoever joins leaves its item's so; in a workspace of unknown contents they are cleared by a
// small kernel in front, beside which this one starts (programmatic launch: 0.6 us on the device, 2 us
// of the host; a memset 4 us).
//
// In a CTA each warp takes its tokens of a unit on its own: it copies their keys and values
// with 16-byte cp.async through its own ring of stages (no CTA barrier), multiplies, and keeps a
// running maximum, sum and output of the softmax in registers (fp32).  The page numbers are
// copied two rings ahead.  The warps join at an item's end, through the stage just used; the copies
// of the next items' units are in flight meanwhile.  Tokens outside the sequence are copied as
// zeros (size 0), never read: infinities and NaN behind a sequence's end have no say.
//
// Measured (bf16 and fp16, in a graph): 131072 tokens x 8 heads x 128 88 us (0.93 of the copy rate), 64
// sequences of up to 8192 x 8 x 128 85 us (0.90), 8 of up to 4096 x 32 x 128 29 us (0.69), 1000 x 8 x 128
// 8.1 us.  The body runs at 0.94 of the rate of a kernel that only reads; before it 2.5 us (lengths, pages,
// first keys: three waits one after another, and code that is not in the SM yet), behind it 1.5 to 5 us
// of joining (more where one item is shared by many CTAs).  Narrower heads are bound by a warp's
// instructions, about 500 cycles for its 16 tokens (32 up to 64 channels) whatever they weigh: 131072
// tokens x 8 x 96 and x 80 92 us (0.67 and 0.56), x 64 53 us (0.78), x 40 58 us (0.44).  A group of more
// than 32 heads (16 above 128 channels) is several items, each of which reads all keys and values: 16
// sequences of 16384 x 1 head x 128 with 32 query heads 48 us, with 64 76 us.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "device_error.cuh"

namespace tileops {
namespace {

constexpr int kMaxCtas = TILEOPS_PAGED_DECODE_COUNTERS;  // four on each of a B200's 148 SMs
constexpr float kNegInf = -__builtin_huge_valf();

struct CacheStrides {
  int64_t page, slot, head;
};

struct DecodeArgs {
  const void *q, *k, *v;
  const int32_t *table, *lens;
  void* o;
  float* lse;
  int* counters;    // [CTA]: how many CTAs have written their sums of the item that it begins
  float2* stats;    // [CTA][2][row]: score the sums are relative to, sum of weights
  // [CTA][2][row][D, of 16 channels each]: weighted sums, of 16 channels the four of a lane's fragment
  // together (2 t, 2 t + 1, 8 + 2 t, 9 + 2 t), so that they are read by 16 bytes.
  float* partial;
  int64_t q_b, q_h;
  CacheStrides ks, vs;
  int64_t table_stride, num_pages;
  int batch, heads, heads_kv, group, dim, page_size, window, blocks;  // blocks of rows a key head
  int part_rows, part_dim;  // rows of an item, at most; D rounded up to 16
  int room;  // tokens that a row of the table has pages for
  FastDivU32 div_page{1};
  float scale;     // log2(e) times the scale, above zero
  uint32_t flip;   // sign bits that q changes, for a scale below zero
  int* err;
};

// ---- the products ----
__device__ __forceinline__ uint32_t smem_at(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldsm(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// bytes 16, or 0: the 16 bytes are zeroed and src is not read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}

// A weight is exp2((s - top) scale), top the largest score so far: the difference is taken before it is
// scaled, so the largest weight is 1 to the bit however large scores are.  (Rounded exponents instead,
// s scale - round(top scale) by one fma, leave the largest weight at 2^r, r up to half a step of top scale:
// from 2^25 on fp16 weights overflow, or all vanish.)  A pair of scores takes two instructions either way.
// Weights go to the second product in the inputs' type, half a step (2^-8 in bf16, 2^-11 in fp16) off
// each; their sum takes them unrounded.  Up to 8 query heads leave rows 8 to 15 of the product's tile free:
// those take what the weights were rounded off by, also in the inputs' type, and a thread, which has rows
// r and r + 8, adds the two up at the end.  The weights are then 2^-16 and 2^-22 off, and it costs nothing:
// no weights of eight rows of padding are made.  More heads would need a second product, 3 to 10% of the
// time, for what is below the output's own rounding.  In fp16 weights are held times 2^15 (the largest is
// 2^15), so that those down to 2^-29 of the largest keep all their bits.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// What a and b were rounded off by in w.
template <typename T>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pack2<T>(a - held.x, b - held.y);
  } else {
    return pack2<T>(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
  }
}
// The rests' part of a sum; none of one that is not finite (a rest of 0 times an infinite value is NaN).
__device__ __forceinline__ float rest_of(float sum, float rests) {
  return fabsf(sum) < -kNegInf ? rests : 0.0f;
}
template <typename T>
__device__ constexpr float kShift = std::is_same<T, __half>::value ? 15.0f : 0.0f;
template <typename T>
__device__ constexpr float kUnshift = std::is_same<T, __half>::value ? 0x1p-15f : 1.0f;

// A sequence's tokens, and units of them.  Tokens are below 2^31, those of the last unit's behind the end
// may not be: sums of them are unsigned.
struct Span {
  uint32_t begin, end;
  int units;
};
template <int UNIT>
__device__ __forceinline__ Span span_of(const DecodeArgs& a, int b) {
  Span s;
  const int end = min(max(a.lens[b], 0), a.room);
  s.end = end;
  s.begin = a.window > 0 ? max(end - a.window, 0) : 0;
  s.units = (s.end - s.begin + UNIT - 1) / UNIT;
  return s;
}

// The row of all units, cut into equal runs: the first `longer` CTAs take size + 1 places, the rest
// size.  An item takes a place for each of its units and one more, behind them, for the time that
// joining its warps takes (about that of a unit, measured).  There are fewer than 2^31 places.
struct Runs {
  uint32_t size, longer;
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * size + min(c, longer); }
  __device__ __forceinline__ uint32_t cta_of(uint32_t place) const {
    const uint32_t head = longer * (size + 1);
    return place < head ? place / (size + 1) : longer + (place - head) / size;
  }
};

// A unit: item (b, head), head counting blocks of rows of key heads, and which unit of it.
struct Unit {
  int b, head, unit;  // b < 0: none
  Span span;
};
struct Cursor {
  Unit u;
  uint32_t place;
  template <int UNIT>
  __device__ __forceinline__ void next(const DecodeArgs& a) {
    ++place;
    if (++u.unit < u.span.units) return;
    ++place;
    u.unit = 0;
    if (++u.head < a.heads_kv * a.blocks) return;
    u.head = 0;
    do {
      if (++u.b >= a.batch) return;
      u.span = span_of<UNIT>(a, u.b);
    } while (u.span.units == 0);
  }
};

// Four channels of a finished row.
template <typename T>
__device__ __forceinline__ void store_row(T* to, float4 v, float all) {
  const float r = all == 0.0f ? 0.0f : 1.0f / all;
  uint2 w;
  if (all == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  w.x = pack2<T>(v.x * r, v.y * r);
  w.y = pack2<T>(v.z * r, v.w * r);
  *reinterpret_cast<uint2*>(to) = w;
}

// What a warp knows of a unit ahead.
struct Looked {
  Unit u;
  uint32_t place;
  bool last;               // the CTA's last one
  int page[32];            // of the warp's tokens in it, where they are inside the sequence
};

// ROWS: query heads that share the keys and values of a unit, 8, 16 or 32 at most.
template <int DP, int ROWS, int WARPS>
struct Layout {
  static constexpr int kTiles = ROWS == 32 ? 2 : 1;            // of 16 rows
  static constexpr int kHalves = ROWS == 8 ? 1 : 2;            // of a tile's rows, that heads have
  static constexpr int kChunks = DP / 8;                       // 16-byte chunks of a row
  static constexpr int kRow = (DP + 63) / 64 * 64;             // elements of a row in shared memory
  // Tokens of a warp in a unit: 8 KB of keys and values and more, for what a unit costs besides.
  static constexpr int kTokens = DP <= 64 ? 32 : 16;
  // Two stages of 8 KB a warp and 12 warps an SM (8 where 16 rows more take the registers): 512 items of up
  // to 8192 tokens x 128 87 us, 88.5 with three stages and 8 warps, 320 items x 64 30.2 and 31.0 (256 items of
  // up to 4096 tokens x 128 28.2 and 28.1); heads of 192 and 256 as they fit.
  static constexpr int kStages = DP > 192 && WARPS == 4 ? 3 : 2;
  static constexpr int kCtasSm = WARPS == 8   ? 1
                                 : WARPS == 4 ? (DP > 128 ? 1 : kTiles == 1 ? 3 : 2)
                                              : (DP <= 192 ? 4 : 3);
  static constexpr int kUnit = WARPS * kTokens;
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kTile = kTokens * kRow;                 // elements of a warp's keys (or values)
  static constexpr int kRows = 16 * kTiles;
  static constexpr size_t kRing = static_cast<size_t>(WARPS) * kStages * 2 * kTile * 2;
  static constexpr size_t kQ = static_cast<size_t>(kRows) * kRow * 2;
  static constexpr size_t kStats = static_cast<size_t>(WARPS) * kRows * 2 * 4;
  static constexpr int kAhead = 2 * kStages;                   // units whose pages are on their way
  static constexpr size_t kUnits = static_cast<size_t>(WARPS) * kAhead * sizeof(Looked);
  static constexpr size_t kBytes = kRing + kQ + kStats + kUnits;
  // Chunk c of row r lies at chunk c ^ (r % 8): the 8 rows of a matrix in 8 different banks.
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    return (r * (kRow / 8) + (c ^ (r & 7))) * 16;
  }
};

// Waits for the end of the kernel that clears the counters (where there is one): before the first
// count, and before the end, so that it has ended when what follows in the stream starts.
__device__ __forceinline__ void behind_clearing() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename T, int DP, int ROWS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (Layout<DP, ROWS, WARPS>::kCtasSm))
    paged_decode(const __grid_constant__ DecodeArgs a) {
  using L = Layout<DP, ROWS, WARPS>;
  constexpr int kThreads = L::kThreads, kUnit = L::kUnit, MT = L::kTiles, kHalves = L::kHalves;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ bool complete;
  T* const q_smem = reinterpret_cast<T*>(smem + L::kRing);
  float2* const stats = reinterpret_cast<float2*>(smem + L::kRing + L::kQ);  // [warp][row]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Looked* const ahead = reinterpret_cast<Looked*>(smem + L::kRing + L::kQ + L::kStats) + warp * L::kAhead;
  const int heads = a.heads_kv * a.blocks;
  // The first of this warp's tokens in a unit.
  auto first_token = [&](const Unit& u) {
    return u.span.begin + static_cast<uint32_t>(u.unit) * kUnit + warp * L::kTokens;
  };

  // ---- places of the call ----
  // By each warp on its own: every lane takes as many sequences, and then the lane whose sequences
  // hold the run's begin has them shared out likewise.
  auto places = [&](int b) {
    const int units = span_of<kUnit>(a, b).units;
    return units ? static_cast<uint32_t>(units + 1) * heads : 0u;
  };
  int from = 0, count = a.batch;  // the sequences in question
  uint32_t mine, upto, total;
  auto scan = [&]() {
    const int per = (count + 31) / 32;
    mine = 0;
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
      const int n = lane * per + i;
      if (n < count) mine += places(from + n);
    }
    upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t v = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += v;
    }
    return per;
  };
  int per = scan();
  total = __shfl_sync(~0u, upto, 31);
  const uint32_t c = blockIdx.x, ctas = min(total, gridDim.x);

  auto without_tokens = [&]() {  // sequences of none; lengths that the table has no room for
    for (int b = c; b < a.batch; b += gridDim.x) {
      if (threadIdx.x == 0 && a.lens[b] > a.room) report_device_error(a.err, kErrBadPage);
      if (span_of<kUnit>(a, b).units) continue;
      for (int64_t n = threadIdx.x; n < static_cast<int64_t>(a.heads) * a.dim; n += kThreads)
        static_cast<T*>(a.o)[static_cast<int64_t>(b) * a.heads * a.dim + n] = Cvt<T>::from_f(0.0f);
      for (int h = threadIdx.x; h < a.heads; h += kThreads)
        a.lse[static_cast<int64_t>(b) * a.heads + h] = kNegInf;
    }
  };
  if (c >= ctas) {
    without_tokens();
    behind_clearing();
    return;
  }
  Runs runs;
  runs.size = total / ctas;
  runs.longer = total - runs.size * ctas;
  const uint32_t u0 = runs.begin(c), u1 = runs.begin(c + 1);

  // ---- the run's first unit ----
  uint32_t before = 0;  // places of the sequences before `from`
#pragma unroll 1
  while (true) {
    const int at = __ffs(__ballot_sync(~0u, before + upto > u0)) - 1;
    before += __shfl_sync(~0u, upto - mine, at);
    from += at * per;
    if (per == 1) break;
    count = min(per, count - at * per);
    per = scan();
  }
  Cursor look;
  look.u.b = from;
  look.u.span = span_of<kUnit>(a, from);
  look.u.head = (u0 - before) / (look.u.span.units + 1);
  look.u.unit = (u0 - before) - look.u.head * (look.u.span.units + 1);
  look.place = u0;
  if (look.u.unit == look.u.span.units) {  // behind an item: on to the next
    --look.u.unit;
    --look.place;
    look.template next<kUnit>(a);
  }
  if (look.place >= u1) {  // a place behind an item and no more
    without_tokens();
    behind_clearing();
    return;
  }

  // The rows of an item, zeros behind them: fetched while the last unit of the item before is multiplied.
  constexpr int kQChunks = (L::kRows * L::kChunks + kThreads - 1) / kThreads;
  uint4 q_next[kQChunks];
  auto fetch_q = [&](const Unit& at) {
    const int h0 = (at.head / a.blocks) * a.group + (at.head % a.blocks) * L::kRows;
    const int rows = min(L::kRows, a.group - (at.head % a.blocks) * L::kRows);
#pragma unroll
    for (int i = 0; i < kQChunks; ++i) {
      const int n = i * kThreads + threadIdx.x, r = n / L::kChunks, ch = n % L::kChunks;
      q_next[i] = make_uint4(0, 0, 0, 0);
      if (r < rows && ch * 8 < a.dim)
        q_next[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at.b * a.q_b +
                                                    (h0 + r) * a.q_h + ch * 8);
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int i = 0; i < kQChunks; ++i) {
      const int n = i * kThreads + threadIdx.x, r = n / L::kChunks, ch = n % L::kChunks;
      const uint4 w = q_next[i];
      if (r < L::kRows)
        *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(q_smem) + L::at(r, ch)) =
            make_uint4(w.x ^ a.flip, w.y ^ a.flip, w.z ^ a.flip, w.w ^ a.flip);
    }
  };
  fetch_q(look.u);

  // ---- copies: the pages of a unit kAhead units ahead, its keys and values kStages ahead ----
  const uint32_t ring = smem_at(smem) + warp * (L::kStages * 2 * L::kTile * 2);
  auto look_up = [&](int slot) {
    Looked& w = ahead[slot];
    Unit u = look.u;
    const uint32_t place = look.place;
    if (look.place >= u1) {
      u.b = -1;
    } else {
      const uint32_t t = first_token(u) + lane;
      if (lane < L::kTokens && t < u.span.end)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(&w.page[lane])),
                     "l"(a.table + u.b * a.table_stride + a.div_page.div(t))
                     : "memory");
      look.template next<kUnit>(a);
    }
    if (lane == 0) {
      w.u = u;
      w.place = place;
      w.last = look.place >= u1;
    }
  };
  auto issue = [&](int stage, int slot) {
    const Looked& w = ahead[slot];
    const Unit u = w.u;
    if (u.b < 0) return;
    const uint32_t t = first_token(u) + lane;
    const int head = u.head / a.blocks;
    const T* k = static_cast<const T*>(a.k) + head * a.ks.head;
    const T* v = static_cast<const T*>(a.v) + head * a.vs.head;
    int64_t k_at = 0, v_at = 0;
    bool inside = lane < L::kTokens && t < u.span.end;
    if (inside) {
      const int page = w.page[lane];
      if (page >= 0 && page < a.num_pages) {
        const int place = static_cast<int>(t - a.div_page.div(t) * a.page_size);
        k_at = page * a.ks.page + place * a.ks.slot;
        v_at = page * a.vs.page + place * a.vs.slot;
      } else {
        report_device_error(a.err, kErrBadPage);
        inside = false;
      }
    }
    const uint32_t rows = __ballot_sync(~0u, inside);
    const uint32_t to = ring + stage * (2 * L::kTile * 2);
    // A row by neighbouring lanes as a whole.  (8 lanes for 128 bytes of a row, 4 rows at a time, take fewer
    // instructions, but where heads lie side by side half rows are fetched apart: 3% longer.)
#pragma unroll
    for (int i = 0; i < L::kTokens * L::kChunks / 32; ++i) {
      const int row = (i * 32 + lane) / L::kChunks, chunk = (i * 32 + lane) % L::kChunks;
      const bool there = ((rows >> row) & 1) && chunk * 8 < a.dim;
      const int64_t ka = __shfl_sync(~0u, k_at, row), va = __shfl_sync(~0u, v_at, row);
      const int64_t col = there ? chunk * 8 : 0;
      copy16(to + L::at(row, chunk), k + ka + col, there ? 16 : 0);
      copy16(to + L::kTile * 2 + L::at(row, chunk), v + va + col, there ? 16 : 0);
    }
  };
#pragma unroll 1
  for (int n = 0; n < L::kStages; ++n) look_up(n);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
#pragma unroll 1
  for (int n = 0; n < L::kStages; ++n) {
    issue(n, n);
    look_up(L::kStages + n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // ---- products ----
  // top: the score that a row's weights are relative to, its largest.
  // Of eight rows, out[..][2] and [3] are the second numbers' part.
  float out[MT][DP / 8][4], top[MT][kHalves], sum[MT][kHalves];
  auto reset = [&]() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[m][n][e] = 0.0f;
#pragma unroll
      for (int r = 0; r < kHalves; ++r) {
        top[m][r] = kNegInf;
        sum[m][r] = 0.0f;
      }
    }
  };
  store_q();
  reset();
  __syncthreads();
  without_tokens();
  behind_clearing();
  bool began = ahead[0].u.unit == 0;  // the item in hand began in this CTA
  int stage = 0, slot = 0;
  const uint32_t q_at = smem_at(q_smem);
#pragma unroll 1
  while (true) {
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
    __syncwarp();
    const Unit get = ahead[slot].u;
    const bool last = ahead[slot].last;
    const bool ended = get.unit + 1 == get.span.units;
    if (ended && !last) fetch_q(ahead[slot + 1 == L::kAhead ? 0 : slot + 1].u);
    const uint32_t keys = ring + stage * (2 * L::kTile * 2), values = keys + L::kTile * 2;
    const uint32_t t0 = first_token(get);
    if (t0 < get.span.end) {
      constexpr int kBlocks = L::kTokens / 16;
      float s[MT][2 * kBlocks][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2 * kBlocks; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t qa[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) ldsm(q_at + L::at(m * 16 + (lane & 15), k * 2 + (lane >> 4)), qa[m]);
#pragma unroll
        for (int t = 0; t < kBlocks; ++t) {
          uint32_t kb[4];
          ldsm(keys + L::at(t * 16 + (lane & 7) + ((lane >> 4) << 3), k * 2 + ((lane >> 3) & 1)), kb);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma<T>(s[m][2 * t], qa[m], kb[0], kb[1]);
            mma<T>(s[m][2 * t + 1], qa[m], kb[2], kb[3]);
          }
        }
      }
      uint32_t w[MT][kBlocks][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (t0 + L::kTokens > get.span.end) {
#pragma unroll
          for (int n = 0; n < 2 * kBlocks; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t0 + n * 8 + (lane & 3) * 2 + (e & 1) >= get.span.end) s[m][n][e] = kNegInf;
        }
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {  // rows lane / 4 and lane / 4 + 8
          float high = kNegInf;
#pragma unroll
          for (int n = 0; n < 2 * kBlocks; ++n)
            high = fmaxf(high, fmaxf(s[m][n][2 * r], s[m][n][2 * r + 1]));
          high = fmaxf(high, __shfl_xor_sync(~0u, high, 1));
          high = fmaxf(high, __shfl_xor_sync(~0u, high, 2));
          const float top_new = fmaxf(high, top[m][r]);
          // A row of nothing but -inf so far: exp2(-inf - 0) = 0, not exp2(-inf + inf).
          const float base = top_new == kNegInf ? 0.0f : top_new;
          const float fade = ex2_approx_f((top[m][r] - base) * a.scale);
          top[m][r] = top_new;
          float add = 0.0f;
#pragma unroll
          for (int n = 0; n < 2 * kBlocks; ++n) {
            const float2 less = fadd2(make_float2(s[m][n][2 * r], s[m][n][2 * r + 1]),
                                      make_float2(-base, -base));
            const float2 t = ffma2(less, make_float2(a.scale, a.scale),
                                   make_float2(kShift<T>, kShift<T>));
            const float w0 = ex2_approx_f(t.x), w1 = ex2_approx_f(t.y);
            add += w0 + w1;
            uint32_t(&to)[4] = w[m][n / 2];
            to[n % 2 * 2 + r] = pack2<T>(w0, w1);
            if constexpr (kHalves == 1) to[n % 2 * 2 + 1] = rest2<T>(w0, w1, to[n % 2 * 2]);
          }
          sum[m][r] = sum[m][r] * fade + add;
          if (__any_sync(~0u, fade != 1.0f)) {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              out[m][n][2 * r] *= fade;
              out[m][n][2 * r + 1] *= fade;
              if (kHalves == 1) {
                out[m][n][2] *= fade;
                out[m][n][3] *= fade;
              }
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
#pragma unroll
        for (int t = 0; t < kBlocks; ++t) {
          uint32_t vb[4];
          ldsm_t(values + L::at(t * 16 + (lane & 15), n * 2 + (lane >> 4)), vb);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma<T>(out[m][2 * n], w[m][t], vb[0], vb[1]);
            mma<T>(out[m][2 * n + 1], w[m][t], vb[2], vb[3]);
          }
        }
      }
    }
    if (ended || last) {
      // ---- the warps' sums of the item, joined through the stage just used ----
      bool whole = began && ended;
      const int block = get.head % a.blocks;
      const int h0 = (get.head / a.blocks) * a.group + block * L::kRows;
      const int rows = min(L::kRows, a.group - block * L::kRows);
#pragma unroll 1
      while (true) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < kHalves; ++r) {
            float v = sum[m][r];
            v += __shfl_xor_sync(~0u, v, 1);
            v += __shfl_xor_sync(~0u, v, 2);
            if ((lane & 3) == 0)
              stats[warp * L::kRows + m * 16 + r * 8 + lane / 4] = make_float2(top[m][r], v);
          }
        unsigned char* const own = smem + (warp * L::kStages + stage) * (2 * L::kTile * 2);
        constexpr int kPad = L::kRow;  // floats of a row there: 16 rows fill the stage
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          __syncwarp();
          // 8-column group n of row r at group (n + r) % groups: the 8 rows in different banks.
#pragma unroll
          for (int r = 0; r < kHalves; ++r) {
            if (m * 16 + r * 8 >= rows) continue;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              const int row = r * 8 + lane / 4;
              const int col = (n + lane / 4) % (DP / 8) * 8 + (lane & 3) * 2;
              float2 v = make_float2(out[m][n][2 * r], out[m][n][2 * r + 1]);
              if (kHalves == 1) {
                v.x += rest_of(v.x, out[m][n][2]);
                v.y += rest_of(v.y, out[m][n][3]);
              }
              *reinterpret_cast<float2*>(own + (row * kPad + col) * 4) = v;
            }
          }
          __syncthreads();
          if (m == 0) store_q();
          for (int n = threadIdx.x; n < min(16, rows - m * 16) * (DP / 4); n += kThreads) {
            const int r = n / (DP / 4), quad = n % (DP / 4), row = m * 16 + r;
            // Four channels in a row for o; of a lane's fragment for other CTAs.
            const int d0 = whole ? quad * 4 : quad / 4 * 16 + quad % 4 * 2, d1 = whole ? d0 + 2 : d0 + 8;
            if (d0 >= a.dim) continue;
            auto at_col = [&](int d) { return (d / 8 + (r & 7)) % (DP / 8) * 8 + d % 8; };
            const int c0 = at_col(d0), c1 = at_col(d1);
            float2 st[WARPS];
            float high = kNegInf;
#pragma unroll
            for (int x = 0; x < WARPS; ++x) {
              st[x] = stats[x * L::kRows + row];
              high = fmaxf(high, st[x].x);
            }
            const float base = high == kNegInf ? 0.0f : high;
            float all = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < WARPS; ++x) {
              const float f = ex2_approx_f((st[x].x - base) * a.scale);
              const float* p = reinterpret_cast<const float*>(
                  smem + (x * L::kStages + stage) * (2 * L::kTile * 2)) + r * kPad;
              const float2 p0 = *reinterpret_cast<const float2*>(p + c0);
              const float2 p1 = *reinterpret_cast<const float2*>(p + c1);
              all += f * st[x].y;
              v.x += f * p0.x;
              v.y += f * p0.y;
              v.z += f * p1.x;
              v.w += f * p1.y;
            }
            if (whole) {
              const int64_t at = static_cast<int64_t>(get.b) * a.heads + h0 + row;
              store_row(static_cast<T*>(a.o) + at * a.dim + d0, v, all);
              if (quad == 0) a.lse[at] = fmaf(base, a.scale, log2f(all * kUnshift<T>));
            } else {
              const int64_t at = (c * 2 + (began ? 1 : 0)) * a.part_rows + row;
              *reinterpret_cast<float4*>(a.partial + at * a.part_dim + quad * 4) = v;
              if (quad == 0) a.stats[at] = make_float2(high, all);
            }
          }
          __syncthreads();
        }
        if (whole) break;
        const uint32_t place = ahead[slot].place;
        const uint32_t owner = began ? c : runs.cta_of(place - get.unit);
        const uint32_t end = ended ? c : runs.cta_of(place + (get.span.units - 1 - get.unit));
        if (threadIdx.x == 0) {  // releases the CTA's sums, written before the barrier
          int count;
          asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
                       : "=r"(count)
                       : "l"(a.counters + owner)
                       : "memory");
          complete = count == static_cast<int>(end - owner);
          if (complete) a.counters[owner] = 0;  // for the next call
        }
        __syncthreads();
        if (!complete) break;
        // The last of the item's CTAs: their sums, shared out to the warps.
        whole = true;
        reset();
#pragma unroll 1
        for (uint32_t x = owner + warp; x <= end; x += WARPS) {
          const int64_t at = (x * 2 + (x == owner)) * a.part_rows;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < kHalves; ++r) {
              const int row = m * 16 + r * 8 + lane / 4;
              if (row >= rows) continue;
              const float2 st = __ldcg(a.stats + at + row);
              const float* p = a.partial + (at + row) * a.part_dim + (lane & 3) * 4;
              float4 v[DP / 16];
#pragma unroll
              for (int n = 0; n < DP / 16; ++n)
                v[n] = n * 16 < a.dim ? __ldcg(reinterpret_cast<const float4*>(p + n * 16))
                                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              const float top_new = fmaxf(top[m][r], st.x);
              const float base = top_new == kNegInf ? 0.0f : top_new;
              const float fade = ex2_approx_f((top[m][r] - base) * a.scale);
              const float f = ex2_approx_f((st.x - base) * a.scale);
              top[m][r] = top_new;
              sum[m][r] = sum[m][r] * fade + ((lane & 3) == 0 ? f * st.y : 0.0f);
#pragma unroll
              for (int n = 0; n < DP / 16; ++n) {
                float(&x)[4] = out[m][2 * n], (&y)[4] = out[m][2 * n + 1];
                x[2 * r] = x[2 * r] * fade + f * v[n].x;
                x[2 * r + 1] = x[2 * r + 1] * fade + f * v[n].y;
                y[2 * r] = y[2 * r] * fade + f * v[n].z;
                y[2 * r + 1] = y[2 * r + 1] * fade + f * v[n].w;
              }
            }
        }
      }
      if (last) break;
      began = true;
      reset();
    } else {
      __syncwarp();
    }
    const int put = slot + L::kStages < L::kAhead ? slot + L::kStages : slot - L::kStages;
    issue(stage, put);
    look_up(slot);
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage = stage + 1 == L::kStages ? 0 : stage + 1;
    slot = slot + 1 == L::kAhead ? 0 : slot + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

__global__ void __launch_bounds__(512) clear_counters(int* counters) {
  asm volatile("griddepcontrol.launch_dependents;");
  for (int n = threadIdx.x; n < kMaxCtas; n += 512) counters[n] = 0;
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
int padded_dim(int64_t dim) {
  return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
}
int rows_of(int64_t group, int dp) { return group > 16 && dp <= 128 ? 32 : 16; }
bool bad_sizes(int64_t batch, int64_t heads, int64_t heads_kv, int64_t dim) {
  return batch < 0 || batch > 0x7fffff || heads < 1 || heads > 4096 || heads_kv < 1 ||
         heads % heads_kv != 0 || dim < 8 || dim > 256 || dim % 8 != 0;
}

// Places of a call at most: of sequences as long as the table has room for.
int64_t places_of(const DecodeArgs& a, int unit) {
  const int64_t seen = a.window ? std::min(a.room, a.window) : a.room;
  return (std::max<int64_t>(1, (seen + unit - 1) / unit) + 1) * a.batch * (a.heads_kv * a.blocks);
}

// Lets the kernel have its shared memory, once on each device (0.5 us a call otherwise).
template <typename T, int DP, int ROWS, int WARPS>
bool opt_in() {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(paged_decode<T, DP, ROWS, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(Layout<DP, ROWS, WARPS>::kBytes)) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// Whether the rows of neighbouring heads lie in the same 128-byte lines: less than a line apart, and
// not in whole lines.
bool share_lines(const DecodeArgs& a, const CacheStrides& s) {
  return a.heads_kv > 1 && std::abs(s.head) < a.dim + 64 && s.head % 64 != 0;
}

template <typename T, int DP, int ROWS, int WARPS>
int launch_tile(const DecodeArgs& a, bool counters_zero, cudaStream_t s) {
  using L = Layout<DP, ROWS, WARPS>;
  // Where heads lie side by side and share 128-byte lines, fewer CTAs: those of neighbouring heads then stay
  // close to each other in the tokens, and a line is fetched once (320 items of 8009 tokens x 80 199 us
  // for 223, x 40 112 for 164; more CTAs are better with whole lines a head, 512 items x 128 85 us for 97, and
  // where heads lie a page apart, 320 items of 8000 tokens x 80 in pages of 7 160 us for 193).
  int ctas_sm = L::kCtasSm;
  if (WARPS == 4 && (share_lines(a, a.ks) || share_lines(a, a.vs))) ctas_sm = std::min(ctas_sm, 2);
  // No more CTAs than there can be places.
  const int64_t grid = std::min<int64_t>(
      {places_of(a, L::kUnit), static_cast<int64_t>(sm_count()) * ctas_sm, kMaxCtas});
  if (!opt_in<T, DP, ROWS, WARPS>()) return TILEOPS_ELAUNCH;
  if (counters_zero) {
    paged_decode<T, DP, ROWS, WARPS><<<static_cast<unsigned>(grid), L::kThreads, L::kBytes, s>>>(a);
    return launch_status();
  }
  clear_counters<<<1, 512, 0, s>>>(a.counters);
  if (int status = launch_status()) return status;
  // Starts once the first kernel has started, and so behind all that came before that one; the
  // CTAs wait for its end before they count.
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(grid));
  config.blockDim = dim3(L::kThreads);
  config.dynamicSmemBytes = L::kBytes;
  config.stream = s;
  config.attrs = &early;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, paged_decode<T, DP, ROWS, WARPS>, a) != cudaSuccess)
    return TILEOPS_ELAUNCH;
  return launch_status();
}

template <typename T, int DP, int ROWS>
int launch_warps(const DecodeArgs& a, bool counters_zero, cudaStream_t s) {
  // Few items are shared by many CTAs each: one CTA of 8 warps an SM, so that there are fewer sums to join
  // (32 items of 32768 tokens x 128 89 us, 93 with CTAs of 4; but 256 items of up to 4096 32 and 29 us).  Many
  // items: smaller CTAs, more of them at different points of an item (512 sequences of up to 256 tokens,
  // 4096 items, CTAs of 2 warps 42 us, of 4 50; 512 items of up to 8192 tokens 87 and 85).
  // Heads of 192 have no room for two CTAs of 4, nor heads of 256 for 8 warps.
  const int64_t items = static_cast<int64_t>(a.batch) * a.heads_kv * a.blocks;
  if constexpr (DP <= 192) {
    if (items <= sm_count()) return launch_tile<T, DP, ROWS, 8>(a, counters_zero, s);
  }
  if constexpr (DP <= 128) {
    if (items <= 4 * sm_count()) return launch_tile<T, DP, ROWS, 4>(a, counters_zero, s);
  }
  if constexpr (DP > 192) {
    if (items <= sm_count()) return launch_tile<T, DP, ROWS, 4>(a, counters_zero, s);
  }
  return launch_tile<T, DP, ROWS, 2>(a, counters_zero, s);
}

template <typename T, int DP>
int launch_rows(const DecodeArgs& a, bool counters_zero, cudaStream_t s) {
  if (a.group <= 8) return launch_warps<T, DP, 8>(a, counters_zero, s);
  if constexpr (DP <= 128) {
    if (rows_of(a.group, DP) == 32) return launch_warps<T, DP, 32>(a, counters_zero, s);
  }
  return launch_warps<T, DP, 16>(a, counters_zero, s);
}

template <typename T>
int launch_type(const DecodeArgs& a, bool counters_zero, cudaStream_t s) {
  switch (padded_dim(a.dim)) {
    case 64: return launch_rows<T, 64>(a, counters_zero, s);
    case 96: return launch_rows<T, 96>(a, counters_zero, s);
    case 128: return launch_rows<T, 128>(a, counters_zero, s);
    case 192: return launch_rows<T, 192>(a, counters_zero, s);
    default: return launch_rows<T, 256>(a, counters_zero, s);
  }
}

constexpr int64_t kCounterBytes = (kMaxCtas * sizeof(int) + 15) / 16 * 16;

}  // namespace
}  // namespace tileops

using namespace tileops;

extern "C" int64_t tileops_paged_decode_workspace_bytes(int64_t heads, int64_t heads_kv,
                                                        int64_t dim) {
  if (bad_sizes(1, heads, heads_kv, dim)) return -1;
  const int64_t group = heads / heads_kv;
  const int64_t rows = std::min<int64_t>(group, rows_of(group, padded_dim(dim)));
  return kCounterBytes + static_cast<int64_t>(kMaxCtas) * 2 * rows * (round16(dim) + 2) * 4;
}

extern "C" int tileops_paged_decode_fwd(
    const void* q, const void* k_cache, const void* v_cache, const int32_t* page_table,
    const int32_t* seq_lens, void* o, float* lse, void* workspace, int64_t batch, int64_t heads,
    int64_t heads_kv, int64_t dim, int64_t num_pages, int64_t page_size, int64_t table_width,
    int64_t table_stride, const int64_t* strides8, int64_t window, int counters_zero, double scale,
    int dtype, void* stream) {
  if (bad_sizes(batch, heads, heads_kv, dim) || num_pages < 0 || num_pages > 0x7fffffffLL ||
      page_size < 1 || page_size > 0x7fffffffLL || table_width < 0 || table_width > 0x7fffffffLL ||
      page_size * table_width > 0x7fffffffLL - 128 || window < 0 || window > 0x7fffffffLL)
    return TILEOPS_EBADSHAPE;
  if (dtype != TILEOPS_DT_F16 && dtype != TILEOPS_DT_BF16) return TILEOPS_EBADDTYPE;
  if (batch == 0) return TILEOPS_OK;
  if (!q || !k_cache || !v_cache || !seq_lens || !o || !lse || !workspace || !strides8 ||
      (table_width && !page_table))
    return TILEOPS_EINVAL;
  for (int n = 0; n < 8; ++n)
    if (strides8[n] % 8 != 0) return TILEOPS_EALIGN;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace) ||
      reinterpret_cast<uintptr_t>(o) % 8 != 0)  // store_row writes 8 bytes
    return TILEOPS_EALIGN;
  DecodeArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.table = page_table;
  a.lens = seq_lens;
  a.o = o;
  a.lse = lse;
  a.counters = static_cast<int*>(workspace);
  a.q_b = strides8[0];
  a.q_h = strides8[1];
  a.ks = {strides8[2], strides8[3], strides8[4]};
  a.vs = {strides8[5], strides8[6], strides8[7]};
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.batch = static_cast<int>(batch);
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.group = static_cast<int>(heads / heads_kv);
  a.dim = static_cast<int>(dim);
  a.page_size = static_cast<int>(page_size);
  a.room = static_cast<int>(page_size * table_width);
  a.window = static_cast<int>(window);
  const int rows = rows_of(a.group, padded_dim(dim));
  a.blocks = (a.group + rows - 1) / rows;
  a.part_rows = std::min(a.group, rows);
  a.part_dim = static_cast<int>(round16(dim));
  a.stats = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + kCounterBytes);
  a.partial = reinterpret_cast<float*>(a.stats + static_cast<int64_t>(kMaxCtas) * 2 * a.part_rows);
  a.div_page = FastDivU32(static_cast<uint32_t>(page_size));
  // Above zero, so that the largest product has the largest weight and one outside the sequence, -inf,
  // none: the sign goes to q, and 0 is fp32's smallest number (scores below 2^127: weights of 1 - 2^-21 and more).
  a.scale = static_cast<float>(std::max(std::abs(scale) * 1.4426950408889634, 0x1p-149));
  a.flip = scale < 0.0 ? 0x80008000u : 0u;
  if (places_of(a, 32) > 0x7fffffffLL) return TILEOPS_EBADSHAPE;
  a.err = device_error_ptr();
  cudaStream_t s = as_stream(stream);
  return dtype == TILEOPS_DT_F16 ? launch_type<__half>(a, counters_zero != 0, s)
                                 : launch_type<__nv_bfloat16>(a, counters_zero != 0, s);
}
