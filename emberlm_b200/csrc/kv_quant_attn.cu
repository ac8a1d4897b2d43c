// Attention over a key/value cache of 4 or 8 bits for a few query rows a key/value head: single tokens, drafts, small
// groups. out = sum_j softmax_j(scale * q . k_j) v_j, over the positions that a row sees.
//
// A block of R <= 8 * NT rows (the query heads of one key/value head times the new tokens) shares the cache rows, which
// are read once. Seven of a CTA's warps take tiles of 2 KB of key codes (16 to 64 positions); the eighth has TMA bring a stage of seven
// tiles with few, large copies (issuing one takes longer than 2 KB take to arrive: a copy a tile fell behind), three stages in shared
// memory. The codes become exact 16-bit floating numbers in registers, in the layout
// that mma.sync wants, without another trip through shared memory:
//   scores   S^T[16 positions, 8 rows] = K Q^T: ldmatrix gives a lane a word of codes of one group and position; which columns meet
//            in which step of the product is free, as long as Q is laid out the same. The codes enter as fp16 numbers, unscaled, a
//            group at a time, and the group's scale joins in fp32 afterwards: that saves half of the shifts of a bfloat16
//            conversion, and fp32 queries keep 22 bits in two fp16 terms (after a power of two has brought the row near 64);
//   softmax  maximum, exponentials and sums in fp32, in the log2 domain; the reference point moves only when a score exceeds it
//            by more than 2^8, so that most tiles need one vote instead of a reduction over the warp;
//   output   O^T[16 columns, 8 rows] += V^T P^T: ldmatrix.trans pairs the codes of two positions, which become c * s in bfloat16; P
//            comes from the scores' fragments by an 8 x 8 transposition (movmatrix). For fp32 outputs it enters as three bfloat16
//            terms (24 bits), for bfloat16 outputs as two: with one, the error of its rounding is as large as the output's own
//            (2.3e-3 of the outputs' size against 1.65e-3). Up to four rows leave half of a tile of eight empty, and the second terms
//            go there (FOLDED): row r + 4 has the query of row r, and so its probabilities, of which it keeps what the first term
//            leaves over; a second product costs 4 to 10 %
//            (32 ragged sequences of up to 32768 of 8 x 128 in 4 bits 168 -> 184 us; in the empty rows 170).
// The floor is the cache's codes and scales, once. All tiles of all blocks lie on one line, which the CTAs cut into equal parts, so
// that one long sequence keeps all SMs busy as a large batch does; blocks that were cut are joined by a second, small kernel.
// Measured (B200, copy bandwidth 6.45 TB/s): 131072 positions of 8 x 64 in 8 bits, four fp32 rows a head, 143 MB: 45 us, 49 % of that
// bandwidth; 32 ragged sequences of up to 32768 of 8 x 128 in 4 bits, two bfloat16 rows a head, 680 MB: 170 us, 62 %; 64
// windows of 1024 in 8 bits, 144 MB: 46 us, 48 %. The bound is latency at low occupancy: with 128 registers a thread there are 3.6 to 3.7
// warps a scheduler, which issue in half of the cycles (ALU pipe 34 to 48 %, tensor pipe 21 to 28 %, DRAM 42 to 45 %); of the
// cycles between two issues of a warp, fixed latencies take 1.3 to 2.0, memory (spilled registers among it) 0.9 to 1.0, a busy math pipe 0.8 to
// 0.9. At 128 registers fp32 rows over 128 columns spill 224 bytes (4 bits) and 32, bfloat16 rows up to 48.
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "kv_quant_attn.h"
#include "mma_bf16.cuh"

namespace ctdk {
namespace kvq {
namespace {

constexpr int kWarps = 7, kStages = 3;   // warps that compute (an eighth one loads: with 128 registers a thread, two CTAs fill an SM)
constexpr int kThreads = (kWarps + 1) * 32;
constexpr float kSlack = 8.0f, kLog2E = 1.4426950408889634f;

template <int D, int BITS>
struct Tile {
  static constexpr int kRow = D * BITS / 8, kScaleRow = D / kGroup * 2;   // bytes of a position
  static constexpr int kKeys = 2048 / kRow;                               // positions of a tile
  static constexpr int kCodes = kKeys * kRow, kScales = kKeys * kScaleRow;
  static constexpr int kBytes = 2 * (kCodes + kScales);                   // that one tile brings
  static constexpr int kBoxes = (kWarps * kKeys + 255) / 256, kBox = kWarps * kKeys / kBoxes;   // copies of a stage (a box is 256 positions at most)
  static_assert(kWarps * kKeys % kBoxes == 0, "equal copies");
  static constexpr int kPitch = D + 4;                                    // floats of a row in the exchange of partial results
  static constexpr int kExchange = kWarps * 8 * kPitch * 4;                // it takes the place of a stage that has been used
  static_assert(kExchange <= kWarps * 2 * (kCodes + kScales), "exchange");
  static constexpr int kStageBytes = (kWarps * kBytes + 1023) / 1024 * 1024;   // (swizzled tiles start at multiples of 1 KB)
  static constexpr int kSmem = 1024 + kStages * kStageBytes;
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same on top of init[0] in the even columns, init[1] in the odd ones.
__device__ __forceinline__ void mma_f16_from(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&init)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(init[0]), "f"(init[1]));
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lds_words(uint32_t (&w)[1], uint32_t a) { asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a)); }
__device__ __forceinline__ void lds_words(uint32_t (&w)[2], uint32_t a) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
}
__device__ __forceinline__ void lds_words(uint32_t (&w)[4], uint32_t a) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
}
// (x, y) as N packed terms, each the rest of the ones before, rounded.
template <int N>
__device__ __forceinline__ void terms_f16(float x, float y, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = pack_f16(x, y);
    if (i + 1 < N) {
      float u, v;
      unpack_f16(t[i], u, v);
      x -= u, y -= v;
    }
  }
}
template <int N>
__device__ __forceinline__ void terms_bf16(float x, float y, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = pack_bf16(x, y);
    if (i + 1 < N) {
      x -= __uint_as_float(t[i] << 16);
      y -= __uint_as_float(t[i] & 0xffff0000u);
    }
  }
}

// N neighbouring values (16 bytes or more, aligned) as floats.
template <int N>
__device__ __forceinline__ void load_row(const float* p, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
}
template <int N>
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + i));
    x[i] = __uint_as_float(v.x << 16), x[i + 1] = __uint_as_float(v.x & 0xffff0000u);
    x[i + 2] = __uint_as_float(v.y << 16), x[i + 3] = __uint_as_float(v.y & 0xffff0000u);
  }
}

struct Span {
  int64_t lo, hi;      // tiles of all units, numbered through
};
// A CTA's place in the list of units (sequence, key/value head): the unit it is at, and where that unit's tiles lie.
struct Unit {
  int b, h;
  int64_t begin, end;
  int64_t pos, count;
  Visit v;
};

struct TokenArgs {
  AttnArgs a;
  int rows;            // T * group, 8 * NT at most
  int split;           // 0: one CTA a unit; 1: equal spans of all tiles
  Patterns bits;
};

// What the loads go by.
struct Feed {
  Unit u;
  int64_t lo, hi;                        // the CTA's tiles
  int64_t left;                          // tiles to come
  int at, end;                           // next one, counted from the unit's first; the unit's tiles that are this CTA's
};
// A stage: n tiles of one unit, one a warp.
struct Stage {
  Unit u;
  int j, n, last;                        // first position; last: it ends the unit's part here
  int plain_lo, plain_hi;                // tiles from position plain_lo to plain_hi are seen whole by every row
};
struct Maps {
  CUtensorMap few[2], all[2];            // codes of keys and of values: boxes of one tile, of as many as one copy takes
};

__device__ __forceinline__ int64_t pos_of(const AttnArgs& a, int b) { return a.pos != nullptr ? static_cast<int64_t>(a.pos[b]) : a.pos_all; }
__device__ __forceinline__ int64_t count_of(const AttnArgs& a, int b) {
  return a.count != nullptr ? min(static_cast<int64_t>(a.count[b]), static_cast<int64_t>(a.T)) : a.T;
}
template <int KEYS>
__device__ __forceinline__ Visit visit(const AttnArgs& a, int b) {
  return visit_of(pos_of(a, b), count_of(a, b), 0, a.T, a.c.capacity, a.window, a.sinks, KEYS);
}
template <int KEYS>
__device__ __forceinline__ void visit_unit(const AttnArgs& a, Unit& u) {
  u.pos = pos_of(a, u.b);
  u.count = count_of(a, u.b);
  u.v = visit_of(u.pos, u.count, 0, a.T, a.c.capacity, a.window, a.sinks, KEYS);
}
// Moves to the next unit that has tiles.
template <int KEYS>
__device__ __forceinline__ void next_unit(const AttnArgs& a, Unit& u) {
  const int64_t n = u.end - u.begin;
  if (++u.h < a.c.Hk) {
    u.begin = u.end;
    u.end += n;
    return;
  }
  u.h = 0;
  do {
    ++u.b;
    visit_unit<KEYS>(a, u);
  } while (u.v.tiles == 0 && u.b + 1 < a.c.B);
  u.begin = u.end;
  u.end += u.v.tiles;
}

__device__ __forceinline__ int64_t span_start(int64_t all, int i, int n) { return quotient(all * i, n); }

// Sum over the CTA of one value a thread (all threads get it), and of the values of the threads before (exclusive).
__device__ __forceinline__ int64_t cta_sum(int64_t x, int64_t* before, int64_t* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) smem[warp] = s;
  __syncthreads();
  int64_t all = 0, pre = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w == warp) pre = all;
    all += smem[w];
  }
  if (before != nullptr) *before = pre + s - x;
  return all;
}

// CTAs that share `all` tiles: no more than get one for each of their warps, so none of them is left without (how many tiles
// there are the host may not know).
__device__ __forceinline__ int sharing(int64_t all, int ctas) {
  const int64_t n = quotient(all + kWarps - 1, kWarps);
  return n < ctas ? static_cast<int>(n) : ctas;
}
// The CTA's part `i` of `n` of all units' tiles, and the unit that holds its first one. False: it has none.
template <int KEYS>
__device__ __forceinline__ bool span_of(const AttnArgs& a, int i, int n, Span& span, Unit& u, int64_t* smem) {
  u = {};
  if (a.pos == nullptr && a.count == nullptr) {
    visit_unit<KEYS>(a, u);
    const int64_t all = static_cast<int64_t>(u.v.tiles) * a.c.B * a.c.Hk;
    n = sharing(all, n);
    if (i >= n) return false;
    span = {span_start(all, i, n), span_start(all, i + 1, n)};
    const int64_t k = quotient(span.lo, u.v.tiles);
    u.b = static_cast<int>(quotient(k, a.c.Hk));
    u.h = static_cast<int>(k - static_cast<int64_t>(u.b) * a.c.Hk);
    u.begin = k * u.v.tiles;
    u.end = u.begin + u.v.tiles;
    return true;
  }
  __shared__ int64_t found[2];
  // Tiles of a chunk of sequences, one a thread; more than one chunk: once for their sum, once more to find the place.
  auto mine = [&](int b0) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    return b < a.c.B ? static_cast<int64_t>(visit<KEYS>(a, b).tiles) * a.c.Hk : 0;
  };
  const int step = static_cast<int>(blockDim.x);
  int64_t x = mine(0), before, all = cta_sum(x, &before, smem);
  for (int b0 = step; b0 < a.c.B; b0 += step) all += cta_sum(mine(b0), nullptr, smem);
  n = sharing(all, n);
  if (i >= n) return false;
  span = {span_start(all, i, n), span_start(all, i + 1, n)};
  int64_t base = 0;
  for (int b0 = 0;;) {
    if (span.lo >= base + before && span.lo < base + before + x) found[0] = b0 + threadIdx.x, found[1] = base + before;
    if (a.c.B <= step) break;
    base += cta_sum(x, &before, smem);
    b0 += step;
    if (span.lo < base || b0 >= a.c.B) break;
    x = mine(b0);
    cta_sum(x, &before, smem);
  }
  __syncthreads();
  u.b = static_cast<int>(found[0]);
  visit_unit<KEYS>(a, u);
  const int64_t h = quotient(span.lo - found[1], u.v.tiles);
  u.h = static_cast<int>(h);
  u.begin = found[1] + h * u.v.tiles;
  u.end = u.begin + u.v.tiles;
  return true;
}

// Floats of a CTA's partial result for one unit: sums [rows][D], then the rows' reference points and denominators.
template <int D, int NT>
struct Part {
  static constexpr int kRows = 8 * NT, kFloats = kRows * (D + 2);
};

template <typename QT, int D, int BITS, int NT, bool FOLDED>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
    kvq_token_kernel(const __grid_constant__ Maps maps, const TokenArgs ta) {
  using TL = Tile<D, BITS>;
  constexpr int KEYS = TL::kKeys, BLOCKS = KEYS / 16, GROUPS = D / kGroup, STEPS = D / 16, ROW = TL::kRow;
  constexpr int NQ = sizeof(QT) == 4 ? 2 : 1, NP = sizeof(QT) == 4 ? 3 : 2;   // terms of a query, of a probability
  constexpr int NB = FOLDED ? 1 : NP;                  // products that the terms of a probability take
  static_assert(!FOLDED || (NT == 1 && NP == 2), "two terms in a tile of eight rows");
  constexpr int SW = GROUPS / 2;                       // words of a position's scales
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages];
  __shared__ Stage stages[kStages];
  __shared__ Feed feed;
  __shared__ Unit first_unit;
  __shared__ __align__(16) uint32_t q_terms[NT][NQ][32][2 * STEPS + 4];   // (rows of odd numbers of 16 bytes: no bank conflicts)
  __shared__ float q_factor[8 * NT], q_more[8 * NT], q_init[8 * NT][GROUPS];
  __shared__ int64_t scan[kWarps + 1];
  __shared__ float row_m[kWarps][8 * NT], row_l[kWarps][8 * NT];
  const AttnArgs& a = ta.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  if (threadIdx.x < kStages) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], kWarps);
  }
  if (threadIdx.x == 0) {
    mbar_fence_init();
    for (int i = 0; i < 2; ++i) {
      tma_prefetch_desc(&maps.few[i]);
      tma_prefetch_desc(&maps.all[i]);
    }
  }
  pdl_launch();
  __syncthreads();
  pdl_wait();

  // This CTA's tiles.
  Span span;
  Unit u = {};
  if (ta.split) {
    if (!span_of<KEYS>(a, blockIdx.x, gridDim.x, span, u, scan)) return;
  } else {
    u.b = static_cast<int>(blockIdx.x) / a.c.Hk;
    u.h = static_cast<int>(blockIdx.x) - u.b * a.c.Hk;
    visit_unit<KEYS>(a, u);
    u.begin = 0;
    u.end = u.v.tiles;
    span.lo = 0;
    span.hi = u.v.tiles;
  }
  const int rows = ta.rows;

  if (threadIdx.x == 0) {
    feed.u = first_unit = u;
    feed.lo = span.lo;
    feed.hi = span.hi;
    feed.left = span.hi - span.lo;
    feed.at = static_cast<int>(span.lo - u.begin);
    feed.end = static_cast<int>(min(u.end, span.hi) - u.begin);
  }
  __syncthreads();
  if (warp == kWarps) {
    // The loading warp runs ahead of the others, over the units' borders.
    Feed& f = feed;
    for (int k = 0; f.left > 0; ++k) {
      const int st = k % kStages;
      if (k >= kStages && !wait_w(&empty[st], (k / kStages + 1) & 1, a.status, 212)) break;
      if (lane == 0) {
        while (f.at >= f.end) {
          f.at -= static_cast<int>(f.u.end - f.u.begin);
          next_unit<KEYS>(a, f.u);
          f.end = static_cast<int>(min(f.u.end, f.hi) - f.u.begin);
        }
        const Visit& v = f.u.v;
        const bool sink = f.at < v.sink_tiles;
        const int n = min((sink ? min(v.sink_tiles, f.end) : f.end) - f.at, kWarps), j = v.tile_at(f.at) * KEYS, bh = f.u.b * a.c.Hk + f.u.h;
        f.at += n;
        f.left -= n;
        Stage& g = stages[st];
        g.u = f.u;
        g.j = j;
        g.n = n;
        g.last = f.at == f.end;
        g.plain_lo = sink || a.window == 0 ? 0 : v.hi_row - a.window;
        g.plain_hi = v.lo_row - KEYS + 1;
        if (sink) g.plain_hi = min(g.plain_hi, a.sinks - KEYS);
        const int64_t sc = (static_cast<int64_t>(bh) * a.c.capacity + j) * GROUPS;
        unsigned char* codes = smem + st * TL::kStageBytes;
        unsigned char* scales = codes + 2 * kWarps * TL::kCodes;
        mbar_expect_tx(&full[st], n * TL::kBytes);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unsigned char* dst = codes + i * kWarps * TL::kCodes;
          if (n == kWarps) {
#pragma unroll
            for (int x = 0; x < kWarps * KEYS; x += TL::kBox) tma_load_3d(dst + x * ROW, &maps.all[i], &full[st], 0, j + x, bh);
          } else {
            for (int x = 0; x < n; ++x) tma_load_3d(dst + x * TL::kCodes, &maps.few[i], &full[st], 0, j + x * KEYS, bh);
          }
          bulk_load(scales + i * kWarps * TL::kScales, a.c.scales[i] + sc, n * TL::kScales, &full[st]);
        }
      }
      __syncwarp();
    }
    return;
  }

  // A lane's row address for ldmatrix (16 rows, two neighbouring chunks of 16 bytes), swizzled as TMA has written it.
  const uint32_t row16 = static_cast<uint32_t>(lane & 15) * ROW;
  const uint32_t lane_at = row16 + ((static_cast<uint32_t>(lane >> 4) * 16u) ^ ((row16 >> 3) & (ROW - 16u)));

  const auto together = []() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); };   // the computing warps
  int used = 0;
  bool ok = true, first = true;
  for (;;) {                                           // one unit after the other
    if (!first) ok = wait_w(&full[used % kStages], (used / kStages) & 1, a.status, 213);   // (the stage names its unit)
    const Unit& unit = first || !ok ? first_unit : stages[used % kStages].u;
    const int ub = unit.b, uh = unit.h, hi_row = unit.v.hi_row;
    const int64_t pos = unit.pos, count = unit.count;
    const bool whole = unit.begin >= feed.lo && unit.end <= feed.hi, last_unit = unit.end >= feed.hi, any = ok && feed.lo < feed.hi;
    float* part = whole ? nullptr : a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (unit.begin < feed.lo ? 0 : 1)) * Part<D, NT>::kFloats;
    // Q: a thread takes four columns of a row, a power of two brings the row's largest value near 64, and the terms go to
    // shared memory in the order in which lanes need them: word 2 ks + i of lane 4 (row mod 8) + tig is b_i of product step ks.
    constexpr int kPer = D / 4, kAtOnce = kWarps * 32 / kPer;   // threads of a row: 16 or 32
#pragma unroll 1
    for (int rr = static_cast<int>(threadIdx.x) / kPer; rr < 8 * NT; rr += kAtOnce) {
      const int n = rr / 8, c4 = static_cast<int>(threadIdx.x) % kPer, r = FOLDED ? rr & 3 : rr;
      float x[4] = {};
      if (r < rows) {
        const int t = r / a.group;
        load_row<4>(static_cast<const QT*>(a.q) + ub * a.batch_stride + static_cast<int64_t>(t) * a.row_stride +
                        static_cast<int64_t>(uh * a.group + (r - t * a.group)) * D + 4 * c4, x);
      }
      float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
      for (int o = 1; o < kPer; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;           // 128: not finite
      int up = most == 0.0f || e == 128 ? 0 : min(6 - e, 126);                     // most * 2^up is in [64, 128), or below; from 2^107 on,
      if (up < -100) up += 8;                                                      // for a smaller factor behind the products, in [2^14, 2^15)
      const float f = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= f;
      float sum = (x[0] + x[1]) + (x[2] + x[3]);       // of a group: eight threads
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((c4 & 7) == 0) q_init[rr][c4 / 8] = sum * (BITS == 4 ? -8.0f * 0x1p-24f : -128.0f * 0x1p-24f);
      if (c4 == 0) {                                   // 2^down, down from -117 to 122 (fp32) or 137; there, what exceeds 2^120 goes to the sums of the codes
        const int down = (NQ == 1 ? 24 : 9) - up, first = NQ == 1 ? min(down, 120) : down;
        q_factor[rr] = fminf(fmaxf(a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + first) << 23), -FLT_MAX), FLT_MAX);   // (scores of zero stay)
        q_more[rr] = __uint_as_float(static_cast<uint32_t>(127 + down - first) << 23);
      }
      if constexpr (BITS == 4) {                       // columns 8 tig + c of a group: pairs (c, c + 4); odd c times 2^-4 beside raw codes
        const int row_lane = (rr & 7) * 4 + ((c4 >> 1) & 3), half = c4 & 1, word = 4 * (c4 >> 3);
        uint32_t t01[NQ], t23[NQ];
        constexpr float odd = NQ == 1 ? 0.0625f : 1.0f;
        terms_f16<NQ>(x[0], x[1] * odd, t01);
        terms_f16<NQ>(x[2], x[3] * odd, t23);
#pragma unroll
        for (int z = 0; z < NQ; ++z) {
          uint16_t* w = reinterpret_cast<uint16_t*>(&q_terms[n][z][row_lane][word]) + half;
          w[0] = static_cast<uint16_t>(t01[z]);
          w[2] = static_cast<uint16_t>(t01[z] >> 16);
          w[4] = static_cast<uint16_t>(t23[z]);
          w[6] = static_cast<uint16_t>(t23[z] >> 16);
        }
      } else {                                         // columns 4 tig + c of a step: pairs of neighbours
        const int row_lane = (rr & 7) * 4 + (c4 & 3), word = 2 * (c4 >> 2);
        uint32_t t01[NQ], t23[NQ];
        terms_f16<NQ>(x[0], x[1], t01);
        terms_f16<NQ>(x[2], x[3], t23);
#pragma unroll
        for (int z = 0; z < NQ; ++z) {
          q_terms[n][z][row_lane][word] = t01[z];
          q_terms[n][z][row_lane][word + 1] = t23[z];
        }
      }
    }
    first = false;
    together();
    uint32_t qf[NT][NQ][2 * STEPS];
    float factor[NT][2], init[NT][GROUPS][2];          // of rows 2 tig, 2 tig + 1: score to log2 domain; what takes the codes' bias off
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int z = 0; z < NQ; ++z)
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i) qf[n][z][i] = q_terms[n][z][lane][i];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        factor[n][c] = q_factor[8 * n + 2 * tig + c];
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) init[n][gr][c] = q_init[8 * n + 2 * tig + c][gr];
      }
    }
    // Rows 2 tig and 2 tig + 1 of tile n: their positions, reference points (log2 domain) and sums.
    int at_row[NT][2];
    float m[NT][2], l[NT][2], o[NT][STEPS][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = FOLDED ? (2 * tig + c) & 3 : 8 * n + 2 * tig + c;
        at_row[n][c] = r < rows ? row_position(pos, count, r / a.group, a.c.capacity) : -1;
        m[n][c] = -INFINITY;
        l[n][c] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][i][c] = 0.0f;
    }

    // One tile; PLAIN: every valid row sees all of it; HUGE: there are queries whose factor is in two parts.
    auto tile = [&](auto plain, auto some_huge, int j0, uint32_t kbase, uint32_t ksc) {
      constexpr bool PLAIN = decltype(plain)::value, HUGE = decltype(some_huge)::value;
      const uint32_t vbase = kbase + kWarps * TL::kCodes, vsc = ksc + kWarps * TL::kScales;
      float s[BLOCKS][NT][4];
      // ---- scores
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
        uint32_t sc[2][SW];
        lds_words(sc[0], ksc + (16 * k + g) * TL::kScaleRow);
        lds_words(sc[1], ksc + (16 * k + 8 + g) * TL::kScaleRow);
        float acc[NT][4];
#pragma unroll
        for (int x = 0; x < ROW / 32; ++x) {           // two chunks of 16 bytes: two groups of 4-bit codes, one of 8-bit codes
          uint32_t w[4];                               // chunk 2 x of positions g, g + 8; chunk 2 x + 1 of both
          ldsm4(w, kbase + k * 16 * ROW + (lane_at ^ (32u * x)));
          // A group is two steps. The tensor cores cut sums off rather than round them, at the size of the sum so far. For bfloat16
          // queries that does not matter: raw codes, on top of what takes their bias off. fp32 queries meet codes without
          // bias, whose sums are smaller, and their small terms go first.
          auto group = [&](int gr, const uint32_t (&f0)[4], const uint32_t (&f1)[4]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (NQ == 1) {
                mma_f16_from(acc[n], f0, qf[n][0][4 * gr], qf[n][0][4 * gr + 1], init[n][gr]);
                mma_f16(acc[n], f1, qf[n][0][4 * gr + 2], qf[n][0][4 * gr + 3]);
              } else {
                const float zero[2] = {0.0f, 0.0f};
                mma_f16_from(acc[n], f0, qf[n][NQ - 1][4 * gr], qf[n][NQ - 1][4 * gr + 1], zero);
                mma_f16(acc[n], f1, qf[n][NQ - 1][4 * gr + 2], qf[n][NQ - 1][4 * gr + 3]);
                mma_f16(acc[n], f0, qf[n][0][4 * gr], qf[n][0][4 * gr + 1]);
                mma_f16(acc[n], f1, qf[n][0][4 * gr + 2], qf[n][0][4 * gr + 3]);
              }
            }
          };
          auto scaled = [&](int gr) {
            const float s0 = __uint_as_float(gr & 1 ? sc[0][gr / 2] & 0xffff0000u : sc[0][gr / 2] << 16);
            const float s1 = __uint_as_float(gr & 1 ? sc[1][gr / 2] & 0xffff0000u : sc[1][gr / 2] << 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (HUGE)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[n][c] *= q_more[8 * n + 2 * tig + (c & 1)];
#pragma unroll
              for (int c = 0; c < 4; ++c) s[k][n][c] = gr == 0 ? acc[n][c] * (c < 2 ? s0 : s1) : fmaf(acc[n][c], c < 2 ? s0 : s1, s[k][n][c]);
            }
          };
          if constexpr (BITS == 4) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t p[4], q[4];
              codes4_f16(w[2 * y], p);
              codes4_f16(w[2 * y + 1], q);
              if constexpr (NQ == 2) {
                unbias4_f16(p, ta.bits);
                unbias4_f16(q, ta.bits);
              }
              const uint32_t f0[4] = {p[0], q[0], p[1], q[1]}, f1[4] = {p[2], q[2], p[3], q[3]};
              group(2 * x + y, f0, f1);
              scaled(2 * x + y);
            }
          } else {
            uint32_t f[2][4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t p[2], q[2];
              codes8_f16(w[2 * y], p);
              codes8_f16(w[2 * y + 1], q);
              if constexpr (NQ == 2) {
                unbias8_f16(p, ta.bits);
                unbias8_f16(q, ta.bits);
              }
              f[y][0] = p[0], f[y][1] = q[0], f[y][2] = p[1], f[y][3] = q[1];
            }
            group(x, f[0], f[1]);
            scaled(x);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[k][n][c] = __fmul_rn(s[k][n][c], factor[n][c & 1]);   // (rounded as its maximum is)
            if (!PLAIN && !sees(at_row[n][c & 1], j0 + 16 * k + g + 8 * (c >> 1), a.window, a.sinks)) s[k][n][c] = -INFINITY;
          }
      }
      // ---- reference points
      bool grow = false;
      float mx[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = s[0][n][c];
#pragma unroll
          for (int k = 0; k < BLOCKS; ++k) x = fmax3(x, s[k][n][c], s[k][n][c + 2]);
          mx[n][c] = x;
          grow |= x > m[n][c] + kSlack;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(mx[n][c], m[n][c]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            const float f = m[n][c] == x ? 1.0f : ex2(m[n][c] - x);
            m[n][c] = x;
            l[n][c] *= f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
              o[n][i][c] *= f;
              o[n][i][c + 2] *= f;
            }
          }
      }
      // ---- output
      float ref[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) ref[n][c] = m[n][c] == -INFINITY ? 0.0f : m[n][c];
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
        uint32_t pf[NT][NB][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = ex2(s[k][n][c] - ref[n][c & 1]);
          l[n][0] += p[0] + p[2];
          l[n][1] += p[1] + p[3];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t tt[NP];
            terms_bf16<NP>(p[2 * hf], p[2 * hf + 1], tt);
            if constexpr (FOLDED) {
              pf[n][0][hf] = movmatrix(tig < 2 ? tt[0] : tt[1]);
            } else {
#pragma unroll
              for (int y = 0; y < NP; ++y) pf[n][y][hf] = movmatrix(tt[y]);
            }
          }
        }
        uint32_t s2[2][GROUPS];                        // scales of positions (2 tig, 2 tig + 1) and (2 tig + 8, 2 tig + 9)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int tok = 16 * k + 2 * tig + 8 * hf;
          uint32_t sc[2 * SW];
          lds_words(sc, vsc + tok * TL::kScaleRow);
          if (!PLAIN) {
            // A probability of zero must not meet a NaN: positions that no row sees count as zeros, and so, here, do
            // groups that are NaN themselves; the rows that see one of those get their NaN below.
#pragma unroll
            for (int i = 0; i < 2 * SW; ++i) {
              if (j0 + tok + i / SW >= hi_row) sc[i] = 0;
              if (is_nan_scale(sc[i])) sc[i] &= 0xffff0000u;
              if (is_nan_scale(sc[i] >> 16)) sc[i] &= 0x0000ffffu;
            }
          }
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) s2[hf][gr] = prmt(sc[gr / 2], sc[SW + gr / 2], gr & 1 ? 0x7632 : 0x5410);
        }
        // (for fp32 outputs the block's sums are formed apart, smallest terms first, and added in fp32: hundreds of sums that are
        // cut off, one on top of the other, cost 1e-5)
        auto product = [&](int i, const uint32_t (&f)[4]) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (NP == 2) {
#pragma unroll
              for (int y = NB - 1; y >= 0; --y) mma_bf16(o[n][i], f, pf[n][y][0], pf[n][y][1]);
            } else {
              float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int y = NP - 1; y >= 0; --y) mma_bf16(t, f, pf[n][y][0], pf[n][y][1]);
              fadd2(o[n][i][0], o[n][i][1], o[n][i][0], o[n][i][1], t[0], t[1]);
              fadd2(o[n][i][2], o[n][i][3], o[n][i][2], o[n][i][3], t[2], t[3]);
            }
          }
        };
#pragma unroll
        for (int x = 0; x < ROW / 32; ++x) {
          uint32_t w[4];                               // chunk 2 x of both pairs of positions, chunk 2 x + 1 of both
          ldsm4_trans(w, vbase + k * 16 * ROW + (lane_at ^ (32u * x)));
          if constexpr (BITS == 4) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {              // a chunk is a group: columns 4 g .. 4 g + 3 of it
              const int gr = 2 * x + y;
              uint32_t p[4], q[4];
              values4_bf16(w[2 * y], s2[0][gr], bias4(s2[0][gr]), ta.bits, p);
              values4_bf16(w[2 * y + 1], s2[1][gr], bias4(s2[1][gr]), ta.bits, q);
              const uint32_t f0[4] = {p[0], p[1], q[0], q[1]}, f1[4] = {p[2], p[3], q[2], q[3]};
              product(2 * gr, f0);
              product(2 * gr + 1, f1);
            }
          } else {
            const Scale8 c0 = scale8(s2[0][x]), c1 = scale8(s2[1][x]);
#pragma unroll
            for (int y = 0; y < 2; ++y) {              // a chunk is half a group: columns 2 g, 2 g + 1 of it
              uint32_t p[2], q[2];
              values8_bf16(w[2 * y], c0, ta.bits, p);
              values8_bf16(w[2 * y + 1], c1, ta.bits, q);
              const uint32_t f[4] = {p[0], p[1], q[0], q[1]};
              product(2 * x + y, f);
            }
          }
        }
      }
      if (!PLAIN) {                                    // NaN groups of values: the rows that see them
        bool nan = false;
        for (int i = lane; i < KEYS * GROUPS; i += 32) nan |= is_nan_scale(lds16(vsc + 2 * i)) && j0 + i / GROUPS < hi_row;
        if (__any_sync(0xffffffffu, nan)) {
#pragma unroll 1
          for (int i = 0; i < KEYS; ++i)
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr)
              if (is_nan_scale(lds16(vsc + i * TL::kScaleRow + gr * 2)))
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int c = 0; c < 2; ++c)
                    if (sees(at_row[n][c], j0 + i, a.window, a.sinks))
#pragma unroll
                      for (int x = 2 * gr; x < 2 * gr + 2; ++x) o[n][x][c] = o[n][x][c + 2] = __int_as_float(0x7fc00000);
        }
      }
    };

    int st = used % kStages, all_ok;
    for (bool more = any; more && ok; ++used) {
      st = used % kStages;
      ok = wait_w(&full[st], (used / kStages) & 1, a.status, 210);
      if (!ok) break;
      const Stage& f = stages[st];
      more = f.last == 0;
      if (warp < f.n) {
        const uint32_t kbase = smem_u32(smem) + st * TL::kStageBytes + warp * TL::kCodes;
        const uint32_t ksc = smem_u32(smem) + st * TL::kStageBytes + 2 * kWarps * TL::kCodes + warp * TL::kScales;
        const int j0 = f.j + warp * KEYS;
        bool huge = false;                             // (by the factors, which are at hand)
        if constexpr (NQ == 1) {
#pragma unroll
          for (int n = 0; n < NT; ++n) huge |= fmaxf(fabsf(factor[n][0]), fabsf(factor[n][1])) > 0x1p105f;
          huge = __any_sync(0xffffffffu, huge);
        }
        if (j0 >= f.plain_lo && j0 <= f.plain_hi && !huge) {
          tile(std::true_type{}, std::false_type{}, j0, kbase, ksc);
        } else if (!huge) {
          tile(std::false_type{}, std::false_type{}, j0, kbase, ksc);
        } else if constexpr (NQ == 1) {
          tile(std::false_type{}, std::true_type{}, j0, kbase, ksc);
        }
      }
      __syncwarp();
      if (lane == 0 && more) mbar_arrive(&empty[st]);  // (the unit's last stage is needed below first)
    }

    // ---- the warps' results of this unit together
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[n][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        if (g == 0) {
          row_m[warp][8 * n + 2 * tig + c] = m[n][c];
          row_l[warp][8 * n + 2 * tig + c] = x;
        }
      }
    // All warps have left the stage st: its room serves for the exchange. (They give up together.)
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, 1, %2, p;\n selp.b32 %0, 1, 0, q;\n}"
                 : "=r"(all_ok) : "r"(static_cast<int>(ok)), "n"(kWarps * 32) : "memory");
    ok = all_ok != 0;
    float* exchange = reinterpret_cast<float*>(smem + st * TL::kStageBytes);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        float* e = exchange + (warp * 8 + 2 * tig) * TL::kPitch + 16 * i + g;
        e[0] = o[n][i][0];
        e[TL::kPitch] = o[n][i][1];
        e[8] = o[n][i][2];
        e[TL::kPitch + 8] = o[n][i][3];
      }
      together();
      for (int i = threadIdx.x; i < 8 * D; i += kWarps * 32) {
        const int r = i / D, e = i % D, rr = 8 * n + r;
        if (rr >= rows) continue;
        float mm = row_m[0][rr];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, row_m[w][rr]);
        const float rf = mm == -INFINITY ? 0.0f : mm;
        float sum = 0.0f, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2(row_m[w][rr] - rf);
          ll += f * row_l[w][rr];
          float x = exchange[(w * 8 + r) * TL::kPitch + e];
          if constexpr (FOLDED) x += exchange[(w * 8 + r + 4) * TL::kPitch + e];
          sum += f * x;
        }
        // the column that lane e & 7 had in half (e >> 3) & 1 of tile e >> 4
        const int ti = e >> 4, gi = e & 7, hf = (e >> 3) & 1;
        const int d = BITS == 4 ? 32 * (ti / 2) + 4 * gi + 2 * (ti & 1) + hf : 16 * ti + 2 * gi + hf;
        if (part != nullptr) {
          part[rr * D + d] = sum;
          if (e == 0) {
            part[8 * NT * D + rr] = mm;
            part[8 * NT * D + 8 * NT + rr] = ll;
          }
        } else {
          const int t = rr / a.group, hg = rr - t * a.group;
          const bool valid = row_position(pos, count, t, a.c.capacity) >= 0;
          store_out(static_cast<QT*>(a.out) + ((static_cast<int64_t>(ub) * a.T + t) * a.H + uh * a.group + hg) * D + d, valid ? sum / ll : 0.0f);
        }
      }
      together();
    }
    if (last_unit || !ok) break;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // copies may write where the exchange was
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
  }
  if (!ok)                                             // copies still on their way
    for (int i = 0; i < kStages; ++i, ++used) wait_w(&full[used % kStages], (used / kStages) & 1, a.status, 211);
}

// Joins the parts of the units that several CTAs worked on, in the order of their positions, and writes zeros for the units that
// have nothing to see. One CTA a unit: the parts' maxima and sums first, all at once, then every output as one sum of
// independent loads (a chain of parts, one after the other, took 60 us for 37 parts of four rows).
constexpr int kJoinThreads = 256, kJoinParts = 128;    // parts whose weights are held at a time
template <typename QT, int D, int BITS, int NT>
__global__ void __launch_bounds__(kJoinThreads) kvq_join_kernel(const TokenArgs ta, int ctas) {
  constexpr int KEYS = Tile<D, BITS>::kKeys, kRows = 8 * NT, kOut = (kRows * D + kJoinThreads - 1) / kJoinThreads;
  __shared__ int64_t scan[kJoinThreads / 32];
  __shared__ float weight[kJoinParts][kRows], part_l[kJoinParts][kRows], row_m[kRows], row_l[kRows];
  const AttnArgs& a = ta.a;
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.x / a.c.Hk, h = blockIdx.x - b * a.c.Hk;
  const int64_t pos = pos_of(a, b), count = count_of(a, b);
  const Visit v = visit<KEYS>(a, b);
  int64_t all, begin;
  if (a.pos == nullptr && a.count == nullptr) {
    all = static_cast<int64_t>(v.tiles) * a.c.B * a.c.Hk;
    begin = static_cast<int64_t>(v.tiles) * blockIdx.x;
  } else {
    int64_t n = 0, before = 0;
    for (int i = threadIdx.x; i < a.c.B; i += kJoinThreads) {
      const int64_t x = visit<KEYS>(a, i).tiles;
      n += x;
      if (i < b) before += x;
    }
    all = cta_sum(n, nullptr, scan) * a.c.Hk;
    begin = cta_sum(before, nullptr, scan) * a.c.Hk + static_cast<int64_t>(v.tiles) * h;
  }
  QT* out = static_cast<QT*>(a.out) + (static_cast<int64_t>(b) * a.T * a.H + h * a.group) * D;
  if (v.tiles == 0) {
    for (int i = threadIdx.x; i < ta.rows * D; i += kJoinThreads) {
      const int r = i / D, t = r / a.group;
      store_out(out + (static_cast<int64_t>(t) * a.H + r - t * a.group) * D + i % D, 0.0f);
    }
    return;
  }
  ctas = sharing(all, ctas);
  const int64_t end = begin + v.tiles;
  const int c0 = static_cast<int>(quotient((begin + 1) * ctas - 1, all)), c1 = static_cast<int>(quotient(end * ctas - 1, all));
  if (c0 == c1) return;
  // The first part is its CTA's last unit, the others are their CTAs' first.
  const float* first = a.part + (static_cast<int64_t>(c0) * 2 + 1) * Part<D, NT>::kFloats;
  auto part_of = [&](int c) { return c == c0 ? first : a.part + static_cast<int64_t>(c) * 2 * Part<D, NT>::kFloats; };
  float sum[kOut];
#pragma unroll
  for (int i = 0; i < kOut; ++i) sum[i] = 0.0f;
  if (threadIdx.x < kRows) {
    row_m[threadIdx.x] = -INFINITY;
    row_l[threadIdx.x] = 0.0f;
  }
  for (int p0 = c0; p0 <= c1; p0 += kJoinParts) {
    const int n = min(kJoinParts, c1 - p0 + 1);
    __syncthreads();
    for (int i = threadIdx.x; i < n * kRows; i += kJoinThreads) {
      const float* p = part_of(p0 + i / kRows) + kRows * D + i % kRows;
      weight[i / kRows][i % kRows] = p[0];
      part_l[i / kRows][i % kRows] = p[kRows];
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float again[NT];                                   // what the sums of earlier parts are multiplied by (rows warp, warp + 8)
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int r = warp + 8 * x;
      float m = row_m[r];
      for (int i = lane; i < n; i += 32) m = fmaxf(m, weight[i][r]);
      m = warp_max(m);
      const float ref = m == -INFINITY ? 0.0f : m;
      float l = 0.0f;
      for (int i = lane; i < n; i += 32) {
        const float w = ex2(weight[i][r] - ref);
        weight[i][r] = w;
        l += w * part_l[i][r];
      }
      l = warp_sum(l);
      again[x] = ex2(row_m[r] - ref);
      __syncwarp();
      if (lane == 0) {
        row_l[r] = row_l[r] * again[x] + l;
        row_m[r] = m;
      }
    }
    if (p0 != c0) {                                    // (more parts than weights are held at a time)
      __shared__ float scale[kRows];
#pragma unroll
      for (int x = 0; x < NT; ++x)
        if (lane == 0) scale[warp + 8 * x] = again[x];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kOut; ++i)
        if (threadIdx.x + i * kJoinThreads < kRows * D) sum[i] *= scale[(threadIdx.x + i * kJoinThreads) / D];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      const int e = threadIdx.x + i * kJoinThreads, r = e / D;
      if (r >= ta.rows) continue;
      int p = 0;
      if (p0 == c0) sum[i] += weight[p++][r] * first[e];
      const float* others = a.part + static_cast<int64_t>(p0 + p) * 2 * Part<D, NT>::kFloats + e;
#pragma unroll 8
      for (; p < n; ++p, others += 2 * Part<D, NT>::kFloats) sum[i] += weight[p][r] * others[0];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOut; ++i) {
    const int e = threadIdx.x + i * kJoinThreads, r = e / D, t = r / a.group;
    if (r >= ta.rows) continue;
    const bool valid = row_position(pos, count, t, a.c.capacity) >= 0;
    store_out(out + (static_cast<int64_t>(t) * a.H + r - t * a.group) * D + e % D, valid ? sum[i] / row_l[r] : 0.0f);
  }
}

// CTAs of the split form: as many as run at a time, fewer where a CTA's warps would not get a tile each.
int split_ctas(int64_t rows, int64_t units, int64_t tiles) {
  const int full = (rows <= 8 ? 2 : 1) * sm_count();
  const int64_t want = (units * tiles + kWarps - 1) / kWarps;
  return static_cast<int>(want < full ? (want < 1 ? 1 : want) : full);
}
int tile_keys(int D, int bits) { return 2048 / (D * bits / 8); }
// Most tiles that a unit can have.
int64_t most_tiles(const AttnArgs& a, int D, int bits) {
  const int keys = tile_keys(D, bits);
  if (a.pos == nullptr) return visit_of(a.pos_all, a.T, 0, a.T, a.c.capacity, a.window, a.sinks, keys).tiles;
  int64_t n = a.c.capacity;
  if (a.window > 0) n = min(n, static_cast<int64_t>(a.window) + a.T + a.sinks + 3 * keys);
  return (n + keys - 1) / keys;
}
// Whether the work is split over all SMs: not where a unit has few tiles, for which the shares' beginnings and the second launch cost more
// than they save. Split and unsplit, us, 8 bits, 8 x 128, two fp32 rows a head: one sequence of 15, 35, 49, 98 tiles 12.4 / 7.2,
// 9.9 / 9.8, 10.5 / 12.2, 12.6 / 20.6; 32 sequences 18.3 / 9.7, 23.1 / 14.2, 25.8 / 17.7, 38.0 / 32.1. The rule asks a unit's tiles alone,
// as it must where positions lie on the device: one long sequence among short ones has to be split. Where all units are known to be
// alike and as many as the CTAs (pos_all, or a window), unsplit would be faster from 36 to some 100 tiles too; the rule does not ask that.
bool split_wanted(int64_t tiles) { return tiles > 5 * kWarps; }

template <typename QT, int D, int BITS, int NT, bool FOLDED = false>
int launch_token(const TokenArgs& ta, int ctas, cudaStream_t s) {
  using TL = Tile<D, BITS>;
  constexpr int kSmem = TL::kSmem;
  auto* kernel = kvq_token_kernel<QT, D, BITS, NT, FOLDED>;
  Maps maps;
  const Cache& c = ta.a.c;
  const uint64_t dims[3] = {TL::kRow, static_cast<uint64_t>(c.capacity), static_cast<uint64_t>(c.B) * c.Hk};
  const uint64_t strides[2] = {TL::kRow, static_cast<uint64_t>(c.capacity) * TL::kRow};
  const uint32_t few[3] = {TL::kRow, TL::kKeys, 1}, all[3] = {TL::kRow, TL::kBox, 1};
  for (int i = 0; i < 2; ++i) {
    int rc = encode_tensor_map_u8(&maps.few[i], c.codes[i], 3, dims, strides, few);
    if (rc == CTDK_OK) rc = encode_tensor_map_u8(&maps.all[i], c.codes[i], 3, dims, strides, all);
    if (rc != CTDK_OK) return rc;
  }
  cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
  if (e == cudaSuccess) e = launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, s, maps, ta);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  if (const int rc = check_launch("kvq_attn"); rc != CTDK_OK || !ta.split) return rc;
  e = launch_pdl(kvq_join_kernel<QT, D, BITS, NT>, dim3(static_cast<unsigned>(ta.a.c.B * ta.a.c.Hk)), dim3(kJoinThreads), 0, s, ta, ctas);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  return check_launch("kvq_attn");
}
template <typename QT, int D, int BITS>
int launch_rows(const TokenArgs& ta, int nt, int ctas, cudaStream_t s) {
  if constexpr (sizeof(QT) == 2)
    if (ta.rows <= 4) return launch_token<QT, D, BITS, 1, true>(ta, ctas, s);
  return nt == 1 ? launch_token<QT, D, BITS, 1>(ta, ctas, s) : launch_token<QT, D, BITS, 2>(ta, ctas, s);
}
template <typename QT>
int launch_any(const TokenArgs& ta, int D, int bits, int nt, int ctas, cudaStream_t s) {
  if (D == 64) return bits == 4 ? launch_rows<QT, 64, 4>(ta, nt, ctas, s) : launch_rows<QT, 64, 8>(ta, nt, ctas, s);
  return bits == 4 ? launch_rows<QT, 128, 4>(ta, nt, ctas, s) : launch_rows<QT, 128, 8>(ta, nt, ctas, s);
}

int64_t part_bytes(int D, int64_t rows) {
  const int nt = rows <= 8 ? 1 : 2;
  return static_cast<int64_t>(sm_count()) * (nt == 1 ? 2 : 1) * 2 * (8 * nt * (D + 2)) * 4;
}

}  // namespace
}  // namespace kvq
}  // namespace ctdk

using namespace ctdk;

extern "C" {

int64_t ctdk_kvq_attn_workspace_bytes(const ctdk_kvq_cache* cache, int64_t T, int H) {
  if (const int rc = kvq::check_cache(cache, "kvq_attn"); rc != CTDK_OK) return rc;
  CTDK_REQUIRE(H > 0 && H % cache->Hk == 0, "kvq_attn: heads must be a multiple of kv heads");
  CTDK_REQUIRE(T >= 0 && T <= INT32_MAX / 2 / H, "kvq_attn: bad T");
  if (T == 0 || cache->B == 0) return 0;
  const int64_t rows = T * (H / cache->Hk);
  return rows <= 16 ? kvq::part_bytes(cache->D, rows) : kvq::attn_tc_bytes(cache->B, cache->Hk, cache->D, rows);
}

int ctdk_kvq_attn(const ctdk_kvq_cache* cache, const void* q, int dtype, int64_t row_stride, int64_t batch_stride, int64_t T, int H,
                  const int32_t* pos, int64_t pos_all, const int32_t* count, int64_t window, int64_t sinks, float scale, void* out,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = kvq::check_cache(cache, "kvq_attn"); rc != CTDK_OK) return rc;
  CTDK_REQUIRE(dtype == CTDK_DTYPE_F32 || dtype == CTDK_DTYPE_BF16, "kvq_attn: dtype must be CTDK_DTYPE_F32 or CTDK_DTYPE_BF16");
  CTDK_REQUIRE(H > 0 && H % cache->Hk == 0, "kvq_attn: heads must be a multiple of kv heads");
  CTDK_REQUIRE(window >= 0 && sinks >= 0, "kvq_attn: window and sinks must not be negative");
  CTDK_REQUIRE(T >= 0 && T <= INT32_MAX / 2 / H, "kvq_attn: bad T");
  CTDK_REQUIRE(pos != nullptr || (pos_all >= 0 && pos_all <= cache->capacity - T), "kvq_attn: %lld positions from %lld on exceed the capacity %lld",
               static_cast<long long>(T), static_cast<long long>(pos_all), static_cast<long long>(cache->capacity));
  CTDK_REQUIRE(std::isfinite(scale * kvq::kLog2E), "kvq_attn: scale must be finite");
  if (T == 0 || cache->B == 0) return CTDK_OK;
  const int64_t unit = dtype == CTDK_DTYPE_F32 ? 4 : 8;   // elements in 16 bytes
  CTDK_REQUIRE(q != nullptr && out != nullptr, "kvq_attn: null pointer");
  CTDK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 && row_stride % unit == 0 &&
                   batch_stride % unit == 0 && row_stride >= 0 && batch_stride >= 0,
               "kvq_attn: q, its strides and out must be multiples of 16 bytes");
  kvq::TokenArgs ta;
  kvq::AttnArgs& a = ta.a;
  a.c = kvq::Cache{{static_cast<const uint8_t*>(cache->k_codes), static_cast<const uint8_t*>(cache->v_codes)},
                   {static_cast<const __nv_bfloat16*>(cache->k_scales), static_cast<const __nv_bfloat16*>(cache->v_scales)},
                   cache->capacity, static_cast<int>(cache->B), cache->Hk};
  a.q = q;
  a.out = out;
  a.row_stride = row_stride;
  a.batch_stride = batch_stride;
  a.pos = pos;
  a.count = count;
  a.pos_all = pos_all;
  a.window = window >= cache->capacity ? 0 : static_cast<int>(window);   // reaches every position
  a.sinks = static_cast<int>(sinks < cache->capacity ? sinks : cache->capacity);
  a.T = static_cast<int>(T);
  a.H = H;
  a.group = H / cache->Hk;
  a.scale_log2 = scale * kvq::kLog2E;
  a.part = static_cast<float*>(workspace);
  a.status = device_status_word();
  if (a.status == nullptr) return fail(CTDK_ELAUNCH, "kvq_attn: no status word");
  const int64_t rows = T * a.group, units = cache->B * cache->Hk;
  // More rows than two tiles of mma.sync take (a third one's sums leave no registers): the prompt kernel, whose tiles have 128. 16 rows here,
  // 20 there, us, 8 heads of 64: one sequence of 2048 positions in 4 bits 25 / 19, eight of 16384 46 / 97.
  if (rows > 16) {
    const int64_t need = kvq::attn_tc_bytes(cache->B, cache->Hk, cache->D, rows);
    CTDK_REQUIRE(need == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= need),
                 "kvq_attn: the workspace needs %lld bytes, 16-byte aligned", static_cast<long long>(need));
    return kvq::attn_tc(a, dtype, cache->bits, cache->D, static_cast<cudaStream_t>(stream));
  }
  ta.rows = static_cast<int>(rows);
  ta.bits = kvq::patterns(cache->bits);
  const int nt = rows <= 8 ? 1 : 2;
  const int64_t tiles = kvq::most_tiles(a, cache->D, cache->bits);
  ta.split = kvq::split_wanted(tiles) ? 1 : 0;
  int64_t ctas = units;
  if (ta.split) {
    CTDK_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                     workspace_bytes >= kvq::part_bytes(cache->D, rows),
                 "kvq_attn: the workspace needs %lld bytes, 16-byte aligned", static_cast<long long>(kvq::part_bytes(cache->D, rows)));
    ctas = kvq::split_ctas(rows, units, tiles);
  }
  CTDK_REQUIRE(units <= INT32_MAX, "kvq_attn: too many rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CTDK_DTYPE_F32 ? kvq::launch_any<float>(ta, cache->D, cache->bits, nt, static_cast<int>(ctas), s)
                                 : kvq::launch_any<__nv_bfloat16>(ta, cache->D, cache->bits, nt, static_cast<int>(ctas), s);
}

}  // extern "C"
