// Attention over a key/value cache of 4 or 8 bits for a few query rows a key/value head: single tokens, drafts, small
// groups. out = sum_j softmax_j(scale * q . k_j) v_j, over the positions that a row sees.
//
// A block of R <= 8 * NT rows (the query heads of one key/value head times the new tokens) shares the cache rows, which
// are read once. Warps work alone, each on tiles of 2 KB of key codes (16 to 64 positions), which bulk copies
// bring into the warp's two stages of shared memory; the codes become exact bfloat16 values in registers, in the layout
// that mma.sync wants, without another trip through shared memory:
//   scores   S^T[16 positions, 8 rows] = K Q^T: a lane takes a quarter of the columns of two positions; which columns meet in
//            which step of the product is free, as long as Q is laid out the same, so a lane's codes are consecutive bytes;
//   softmax  maximum, exponentials and sums in fp32, in the log2 domain; the reference point moves only when a score exceeds it
//            by more than 2^8, so that most tiles need one vote instead of a reduction over the warp;
//   output   O^T[16 columns, 8 rows] += V^T P^T: V's fragments pair the codes of two positions (byte permutes), P comes from the
//            scores' fragments by an 8 x 8 transposition (movmatrix).
// fp32 queries and, for fp32 outputs, the probabilities enter as two bfloat16 terms: what that leaves out, at most 2^-16 of a
// term (2^-18 on average), is within the bound of rounding an fp32 sum of 256 terms.
#include <climits>

#include "kv_quant_attn.h"
#include "mma_bf16.cuh"

namespace ctdk {
namespace kvq {
namespace {

constexpr int kWarps = 8, kStages = 2;
constexpr float kSlack = 8.0f;

template <int D, int BITS>
struct Tile {
  static constexpr int kRow = D * BITS / 8, kScaleRow = D / kGroup * 2;   // bytes of a position
  static constexpr int kKeys = 2048 / kRow;                               // positions of a tile
  static constexpr int kCodes = kKeys * kRow, kScales = kKeys * kScaleRow;
  static constexpr int kStage = 2 * (kCodes + kScales);                   // key codes, value codes, key scales, value scales
  static constexpr int kPitch = D + 4;                                    // floats of a row in the exchange of partial results
  static constexpr int kExchange = kWarps * 8 * kPitch * 4;
  static constexpr int kSmem = kWarps * kStages * kStage + kExchange;
};

// Row m of a block of 16 positions holds position place(m): neighbours in m differ in parity, and so do m and m + 2, which
// keeps the keys' and the values' reads of 64-byte rows off each other's banks.
__device__ __forceinline__ int place(int m) { return m ^ ((m >> 1) & 1); }

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t a) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "words");
  if constexpr (N == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
  if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  if constexpr (N >= 4)
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(a + 4 * i));
}

struct Span {
  int64_t lo, hi;      // tiles of all units, numbered through
};
// A CTA's place in the list of units (sequence, key/value head): the unit it is at, and where that unit's tiles lie.
struct Unit {
  int b, h;
  int64_t begin, end;
  Visit v;
};

struct TokenArgs {
  AttnArgs a;
  int rows;            // T * group
  int split;           // 0: one CTA a unit (and a block of 8 * NT rows); 1: equal spans of all tiles
};

__device__ __forceinline__ int64_t pos_of(const AttnArgs& a, int b) { return a.pos != nullptr ? static_cast<int64_t>(a.pos[b]) : a.pos_all; }
__device__ __forceinline__ int64_t count_of(const AttnArgs& a, int b) {
  return a.count != nullptr ? min(static_cast<int64_t>(a.count[b]), static_cast<int64_t>(a.T)) : a.T;
}
template <int KEYS>
__device__ __forceinline__ Visit visit(const AttnArgs& a, int b, int t0, int rows) {
  return visit_of(pos_of(a, b), count_of(a, b), t0, rows, a.c.capacity, a.window, a.sinks, KEYS);
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
    u.v = visit<KEYS>(a, u.b, 0, a.T);
  } while (u.v.tiles == 0 && u.b + 1 < a.c.B);
  u.begin = u.end;
  u.end += u.v.tiles;
}

__device__ __forceinline__ int64_t span_start(int64_t all, int i, int n) { return all * i / n; }

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

// Tiles of all sequences' units.
template <int KEYS>
__device__ __forceinline__ int64_t all_tiles(const AttnArgs& a, int64_t* smem) {
  if (a.pos == nullptr && a.count == nullptr) return static_cast<int64_t>(visit<KEYS>(a, 0, 0, a.T).tiles) * a.c.B * a.c.Hk;
  int64_t n = 0;
  for (int b = threadIdx.x; b < a.c.B; b += blockDim.x) n += visit<KEYS>(a, b, 0, a.T).tiles;
  return cta_sum(n, nullptr, smem) * a.c.Hk;
}

// The unit that holds tile x (x < all tiles).
template <int KEYS>
__device__ __forceinline__ Unit unit_at(const AttnArgs& a, int64_t x, int64_t* smem) {
  Unit u;
  if (a.pos == nullptr && a.count == nullptr) {
    u.v = visit<KEYS>(a, 0, 0, a.T);
    const int64_t n = x / u.v.tiles;
    u.b = static_cast<int>(n / a.c.Hk);
    u.h = static_cast<int>(n % a.c.Hk);
    u.begin = n * u.v.tiles;
    u.end = u.begin + u.v.tiles;
    return u;
  }
  __shared__ int64_t found[2];
  int64_t base = 0;
  for (int b0 = 0;; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const int64_t n = b < a.c.B ? static_cast<int64_t>(visit<KEYS>(a, b, 0, a.T).tiles) * a.c.Hk : 0;
    int64_t before;
    const int64_t sum = cta_sum(n, &before, smem);
    before += base;
    if (x >= before && x < before + n) found[0] = b, found[1] = before;
    base += sum;
    __syncthreads();
    if (x < base || b0 + static_cast<int>(blockDim.x) >= a.c.B) break;
  }
  u.b = static_cast<int>(found[0]);
  u.v = visit<KEYS>(a, u.b, 0, a.T);
  const int64_t h = (x - found[1]) / u.v.tiles;
  u.h = static_cast<int>(h);
  u.begin = found[1] + h * u.v.tiles;
  u.end = u.begin + u.v.tiles;
  return u;
}

__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Floats of a CTA's partial result for one unit: sums [rows][D], then the rows' reference points and denominators.
template <int D, int NT>
struct Part {
  static constexpr int kRows = 8 * NT, kFloats = kRows * (D + 2);
};

template <typename QT, int D, int BITS, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) kvq_token_kernel(const TokenArgs ta) {
  using TL = Tile<D, BITS>;
  constexpr int KEYS = TL::kKeys, BLOCKS = KEYS / 16;
  constexpr bool kSplitQ = sizeof(QT) == 4;            // two bfloat16 terms
  constexpr int NS = kSplitQ ? 2 : 1;
  constexpr int KW = TL::kRow / 16, VW = TL::kRow / 32;   // words of a lane's share of a position: a quarter of the keys', an eighth of the values'
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t bars[kWarps * kStages];
  __shared__ int64_t scan[kWarps];
  __shared__ float row_m[kWarps][8 * NT], row_l[kWarps][8 * NT];
  const AttnArgs& a = ta.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
  if (threadIdx.x < kWarps * kStages) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) mbar_fence_init();
  pdl_launch();
  __syncthreads();
  pdl_wait();

  // This CTA's tiles.
  Span span;
  Unit u = {};
  int r0 = 0;                                          // first row of the block of rows
  if (ta.split) {
    const int64_t all = all_tiles<KEYS>(a, scan);
    span.lo = span_start(all, blockIdx.x, gridDim.x);
    span.hi = span_start(all, blockIdx.x + 1, gridDim.x);
    if (span.lo >= span.hi) return;
    u = unit_at<KEYS>(a, span.lo, scan);
  } else {
    const int blocks = (ta.rows + 8 * NT - 1) / (8 * NT);
    const int64_t id = blockIdx.x, bh = id / blocks;
    r0 = static_cast<int>(id - bh * blocks) * 8 * NT;
    u.b = static_cast<int>(bh / a.c.Hk);
    u.h = static_cast<int>(bh - static_cast<int64_t>(u.b) * a.c.Hk);
    const int t0 = r0 / a.group, t1 = (min(r0 + 8 * NT, ta.rows) - 1) / a.group;
    u.v = visit<KEYS>(a, u.b, t0, t1 - t0 + 1);
    u.begin = 0;
    u.end = u.v.tiles;
    span.lo = 0;
    span.hi = u.v.tiles;
  }
  const int rows = min(8 * NT, ta.rows - r0);

  unsigned char* mine = smem + warp * kStages * TL::kStage;
  uint64_t* bar = &bars[warp * kStages];
  float* exchange = reinterpret_cast<float*>(smem + kWarps * kStages * TL::kStage);

  // Loads run ahead of the products, over the units' borders.
  Unit lu = u;
  int64_t load_at = span.lo + warp;
  int loaded = 0;
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  auto load = [&]() {
    if (load_at >= span.hi) return;
    while (load_at >= lu.end) next_unit<KEYS>(a, lu);
    if (lane == 0) {
      const int64_t j = (static_cast<int64_t>(lu.b) * a.c.Hk + lu.h) * a.c.capacity + static_cast<int64_t>(lu.v.tile_at(static_cast<int>(load_at - lu.begin))) * KEYS;
      unsigned char* dst = mine + (loaded % kStages) * TL::kStage;
      uint64_t* full = &bar[loaded % kStages];
      mbar_expect_tx(full, TL::kStage);
      bulk_load(dst, a.c.codes[0] + j * TL::kRow, TL::kCodes, full, policy);
      bulk_load(dst + 2 * TL::kCodes, a.c.scales[0] + j * (D / kGroup), TL::kScales, full, policy);
      bulk_load(dst + TL::kCodes, a.c.codes[1] + j * TL::kRow, TL::kCodes, full, policy);
      bulk_load(dst + 2 * TL::kCodes + TL::kScales, a.c.scales[1] + j * (D / kGroup), TL::kScales, full, policy);
    }
    ++loaded;
    load_at += kWarps;
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) load();

  int used = 0;
  bool ok = true;
  int64_t at = span.lo + warp;
  for (int64_t seg = span.lo;;) {                      // one unit after the other
    const int64_t seg_end = min(u.end, span.hi);
    const int64_t pos = pos_of(a, u.b), count = count_of(a, u.b);
    // Q's fragments: column (a row of queries) g of tile n; b0, b1 of product step ks in the lane's own order of columns.
    uint32_t qf[NT][D / 16][NS][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + 8 * n + g, t = r / a.group;
      const bool live = 8 * n + g < rows;
      const QT* src = static_cast<const QT*>(a.q) + u.b * a.batch_stride + static_cast<int64_t>(t) * a.row_stride +
                      static_cast<int64_t>(u.h * a.group + (r - t * a.group)) * D + tig * (D / 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        int d[4];
        if (BITS == 4) {                               // words of eight codes: two steps, pairs (c, c + 4)
          const int w = 8 * (ks / 2) + 2 * (ks & 1);
          d[0] = w, d[1] = w + 4, d[2] = w + 1, d[3] = w + 5;
        } else {
          d[0] = 4 * ks, d[1] = 4 * ks + 1, d[2] = 4 * ks + 2, d[3] = 4 * ks + 3;
        }
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = live ? static_cast<float>(src[d[i]]) : 0.0f;
        if constexpr (kSplitQ) {
          split_bf16x2(x[0], x[1], qf[n][ks][0][0], qf[n][ks][1][0]);
          split_bf16x2(x[2], x[3], qf[n][ks][0][1], qf[n][ks][1][1]);
        } else {
          qf[n][ks][0][0] = pack_bf16(x[0], x[1]);
          qf[n][ks][0][1] = pack_bf16(x[2], x[3]);
        }
      }
    }
    // Rows 2 tig and 2 tig + 1 of tile n: their positions, reference points (log2 domain) and sums.
    int at_row[NT][2];
    float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * n + 2 * tig + c;
        at_row[n][c] = r < rows ? row_position(pos, count, (r0 + r) / a.group, a.c.capacity) : -1;
        m[n][c] = -INFINITY;
        l[n][c] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][i][c] = 0.0f;
    }

    for (; at < seg_end; at += kWarps) {
      const int j0 = u.v.tile_at(static_cast<int>(at - u.begin)) * KEYS;
      const int stage = used % kStages;
      ok = ok && mbar_wait_bounded_w(&bar[stage], (used / kStages) & 1, a.status, 210);
      if (!ok) break;
      const uint32_t base = smem_u32(mine + stage * TL::kStage), vbase = base + TL::kCodes;
      const uint32_t ksc = base + 2 * TL::kCodes, vsc = ksc + TL::kScales;
      // every valid row sees every position of most tiles
      const bool plain = j0 + KEYS - 1 <= u.v.lo_row && (a.window == 0 || u.v.hi_row - 1 - j0 < a.window || j0 + KEYS <= a.sinks);
      float s[BLOCKS][NT][4];
      // ---- scores
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
        uint32_t w[2][KW], s2[2], b2[2];
        float sf[2], bf[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int tok = 16 * k + place(g + 8 * hf);
          lds_words(w[hf], base + tok * TL::kRow + tig * (TL::kRow / 4));
          const uint32_t sc = lds16(ksc + tok * TL::kScaleRow + (tig * (D / 4) / kGroup) * 2);
          if (BITS == 4) {
            s2[hf] = prmt(sc, 0, 0x1010);
            b2[hf] = bias4(s2[hf]);
          } else {
            sf[hf] = __uint_as_float(sc << 16);
            bf[hf] = bias8(sf[hf]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[k][n][c] = 0.0f;
        float lo[NT][4] = {};
#pragma unroll
        for (int x = 0; x < KW; ++x) {
          uint32_t f[2][4];
          if constexpr (BITS == 4) {
            f[0][0] = value4<0>(w[0][x], s2[0], b2[0]), f[0][1] = value4<0>(w[1][x], s2[1], b2[1]);
            f[0][2] = value4<1>(w[0][x], s2[0], b2[0]), f[0][3] = value4<1>(w[1][x], s2[1], b2[1]);
            f[1][0] = value4<2>(w[0][x], s2[0], b2[0]), f[1][1] = value4<2>(w[1][x], s2[1], b2[1]);
            f[1][2] = value4<3>(w[0][x], s2[0], b2[0]), f[1][3] = value4<3>(w[1][x], s2[1], b2[1]);
          } else {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              f[0][hf] = values8(magic8<0>(w[hf][x]), magic8<1>(w[hf][x]), sf[hf], sf[hf], bf[hf], bf[hf]);
              f[0][2 + hf] = values8(magic8<2>(w[hf][x]), magic8<3>(w[hf][x]), sf[hf], sf[hf], bf[hf], bf[hf]);
            }
          }
#pragma unroll
          for (int y = 0; y < (BITS == 4 ? 2 : 1); ++y) {
            const int ks = BITS == 4 ? 2 * x + y : x;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16(s[k][n], f[y], qf[n][ks][0][0], qf[n][ks][0][1]);
              if constexpr (kSplitQ) mma_bf16(lo[n], f[y], qf[n][ks][NS - 1][0], qf[n][ks][NS - 1][1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[k][n][c] = (s[k][n][c] + lo[n][c]) * a.scale_log2;
            if (!plain && !sees(at_row[n][c & 1], j0 + 16 * k + place(g + 8 * (c >> 1)), a.window, a.sinks)) s[k][n][c] = -INFINITY;
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
            for (int i = 0; i < D / 16; ++i) {
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
        uint32_t pf[NT][NS][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = ex2(s[k][n][c] - ref[n][c & 1]);
          l[n][0] += p[0] + p[2];
          l[n][1] += p[1] + p[3];
          if constexpr (kSplitQ) {
            split_bf16x2(p[0], p[1], pf[n][0][0], pf[n][NS - 1][0]);
            split_bf16x2(p[2], p[3], pf[n][0][1], pf[n][NS - 1][1]);
          } else {
            pf[n][0][0] = pack_bf16(p[0], p[1]);
            pf[n][0][1] = pack_bf16(p[2], p[3]);
          }
#pragma unroll
          for (int x = 0; x < NS; ++x) {
            pf[n][x][0] = movmatrix(pf[n][x][0]);
            pf[n][x][1] = movmatrix(pf[n][x][1]);
          }
        }
        uint32_t w[4][VW], sc[4];                      // positions 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9 of the block
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m16 = 2 * tig + (i & 1) + 8 * (i >> 1), tok = 16 * k + place(m16);
          lds_words(w[i], vbase + tok * TL::kRow + g * (TL::kRow / 8));
          sc[i] = lds16(vsc + tok * TL::kScaleRow + (g * (D / 8) / kGroup) * 2);
          if (!plain) {
            // A probability of zero must not meet a NaN: positions that no row sees count as zeros, and so, here, do
            // groups that are NaN themselves; the rows that see one of those get their NaN below.
            if (j0 + tok >= u.v.hi_row || is_nan_scale(sc[i])) sc[i] = 0;
          }
        }
        uint32_t s2[2], b2[2];
        float sf[4], bf[4];
        if (BITS == 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s2[i] = prmt(sc[2 * i], sc[2 * i + 1], 0x5410);
            b2[i] = bias4(s2[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sf[i] = __uint_as_float(sc[i] << 16);
            bf[i] = bias8(sf[i]);
          }
        }
        auto product = [&](int i, const uint32_t (&f)[4]) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < NS; ++x) mma_bf16(o[n][i], f, pf[n][x][0], pf[n][x][1]);
        };
#pragma unroll
        for (int x = 0; x < VW; ++x) {
          if constexpr (BITS == 4) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {              // halves of the words: codes 4 y .. 4 y + 3 of both positions
              const uint32_t e = prmt(w[0][x], w[1][x], y ? 0x7632 : 0x5410), f = prmt(w[2][x], w[3][x], y ? 0x7632 : 0x5410);
              const uint32_t f0[4] = {value4<0>(e, s2[0], b2[0]), value4<1>(e, s2[0], b2[0]), value4<0>(f, s2[1], b2[1]), value4<1>(f, s2[1], b2[1])};
              const uint32_t f1[4] = {value4<2>(e, s2[0], b2[0]), value4<3>(e, s2[0], b2[0]), value4<2>(f, s2[1], b2[1]), value4<3>(f, s2[1], b2[1])};
              product(4 * x + 2 * y, f0);
              product(4 * x + 2 * y + 1, f1);
            }
          } else {
            const uint32_t f0[4] = {values8(magic8<0>(w[0][x]), magic8<0>(w[1][x]), sf[0], sf[1], bf[0], bf[1]),
                                    values8(magic8<1>(w[0][x]), magic8<1>(w[1][x]), sf[0], sf[1], bf[0], bf[1]),
                                    values8(magic8<0>(w[2][x]), magic8<0>(w[3][x]), sf[2], sf[3], bf[2], bf[3]),
                                    values8(magic8<1>(w[2][x]), magic8<1>(w[3][x]), sf[2], sf[3], bf[2], bf[3])};
            const uint32_t f1[4] = {values8(magic8<2>(w[0][x]), magic8<2>(w[1][x]), sf[0], sf[1], bf[0], bf[1]),
                                    values8(magic8<3>(w[0][x]), magic8<3>(w[1][x]), sf[0], sf[1], bf[0], bf[1]),
                                    values8(magic8<2>(w[2][x]), magic8<2>(w[3][x]), sf[2], sf[3], bf[2], bf[3]),
                                    values8(magic8<3>(w[2][x]), magic8<3>(w[3][x]), sf[2], sf[3], bf[2], bf[3])};
            product(2 * x, f0);
            product(2 * x + 1, f1);
          }
        }
      }
      if (!plain) {                                    // NaN groups of values: the rows that see them
        bool nan = false;
        for (int i = lane; i < KEYS * (D / kGroup); i += 32) nan |= is_nan_scale(lds16(vsc + 2 * i)) && j0 + i / (D / kGroup) < u.v.hi_row;
        if (__any_sync(0xffffffffu, nan)) {
          for (int i = 0; i < KEYS; ++i)
            if (is_nan_scale(lds16(vsc + i * TL::kScaleRow + (g * (D / 8) / kGroup) * 2)))
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (sees(at_row[n][c], j0 + i, a.window, a.sinks))
#pragma unroll
                    for (int x = 0; x < D / 16; ++x) o[n][x][c] = o[n][x][c + 2] = __int_as_float(0x7fc00000);
        }
      }
      __syncwarp();
      ++used;
      load();
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
    const bool whole = u.begin >= span.lo && u.end <= span.hi;
    float* part = nullptr;
    if (!whole) part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (u.begin < span.lo ? 0 : 1)) * Part<D, NT>::kFloats;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        float* e = exchange + (warp * 8 + 2 * tig) * TL::kPitch + 16 * i + g;
        e[0] = o[n][i][0];
        e[TL::kPitch] = o[n][i][1];
        e[8] = o[n][i][2];
        e[TL::kPitch + 8] = o[n][i][3];
      }
      __syncthreads();
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
          sum += f * exchange[(w * 8 + r) * TL::kPitch + e];
        }
        // column of slot e: tile i of 16 holds columns 2 i and 2 i + 1 of each eighth of the head
        const int gi = e & 7, d = gi * (D / 8) + 2 * (e >> 4) + ((e >> 3) & 1);
        if (part != nullptr) {
          part[rr * D + d] = sum;
          if (e == 0) {
            part[8 * NT * D + rr] = mm;
            part[8 * NT * D + 8 * NT + rr] = ll;
          }
        } else {
          const int t = (r0 + rr) / a.group, hg = (r0 + rr) - t * a.group;
          const bool valid = row_position(pos, count, t, a.c.capacity) >= 0;
          store_out(static_cast<QT*>(a.out) + ((static_cast<int64_t>(u.b) * a.T + t) * a.H + u.h * a.group + hg) * D + d, valid ? sum / ll : 0.0f);
        }
      }
      __syncthreads();
    }
    seg = seg_end;
    if (seg >= span.hi) break;
    next_unit<KEYS>(a, u);
  }
  for (; !ok && used < loaded; ++used) mbar_wait_bounded_w(&bar[used % kStages], (used / kStages) & 1, a.status, 211);   // copies still on their way
}

// Joins the parts of the units that several CTAs worked on, in the order of their positions, and writes zeros for the units that
// have nothing to see.
template <typename QT, int D, int BITS, int NT>
__global__ void __launch_bounds__(D) kvq_join_kernel(const TokenArgs ta, int ctas) {
  constexpr int KEYS = Tile<D, BITS>::kKeys;
  __shared__ int64_t scan[D / 32];
  const AttnArgs& a = ta.a;
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.x / a.c.Hk, h = blockIdx.x - b * a.c.Hk;
  const Visit v = visit<KEYS>(a, b, 0, a.T);
  int64_t all, begin;
  if (a.pos == nullptr && a.count == nullptr) {
    all = static_cast<int64_t>(v.tiles) * a.c.B * a.c.Hk;
    begin = static_cast<int64_t>(v.tiles) * blockIdx.x;
  } else {
    int64_t n = 0, before = 0;
    for (int i = threadIdx.x; i < a.c.B; i += D) {
      const int64_t x = visit<KEYS>(a, i, 0, a.T).tiles;
      n += x;
      if (i < b) before += x;
    }
    all = cta_sum(n, nullptr, scan) * a.c.Hk;
    begin = cta_sum(before, nullptr, scan) * a.c.Hk + static_cast<int64_t>(v.tiles) * h;
  }
  const int d = threadIdx.x;
  QT* out = static_cast<QT*>(a.out) + (static_cast<int64_t>(b) * a.T * a.H + h * a.group) * D + d;
  if (v.tiles == 0) {
    for (int r = 0; r < ta.rows; ++r) store_out(out + (static_cast<int64_t>(r / a.group) * a.H + r % a.group) * D, 0.0f);
    return;
  }
  const int64_t end = begin + v.tiles;
  const int c0 = static_cast<int>(((begin + 1) * ctas - 1) / all), c1 = static_cast<int>((end * ctas - 1) / all);
  if (c0 == c1) return;
  const int64_t pos = pos_of(a, b), count = count_of(a, b);
  for (int r = 0; r < ta.rows; ++r) {
    const int t = r / a.group;
    float x = 0.0f;
    if (row_position(pos, count, t, a.c.capacity) >= 0) {
      float m = -INFINITY, l = 0.0f, s = 0.0f;
      for (int c = c0; c <= c1; ++c) {
        const float* p = a.part + (static_cast<int64_t>(c) * 2 + (begin < span_start(all, c, ctas) ? 0 : 1)) * Part<D, NT>::kFloats;
        const float pm = p[8 * NT * D + r], pl = p[8 * NT * D + 8 * NT + r], ps = p[r * D + d];
        const float nm = fmaxf(m, pm), ref = nm == -INFINITY ? 0.0f : nm, f = ex2(m - ref), e = ex2(pm - ref);
        l = l * f + pl * e;
        s = s * f + ps * e;
        m = nm;
      }
      x = s / l;
    }
    store_out(out + (static_cast<int64_t>(t) * a.H + r % a.group) * D, x);
  }
}

// CTAs of the split form: as many as run at a time, fewer where a CTA's warps would not get a tile each.
int split_ctas(int D, int bits, int64_t rows, int64_t units, int64_t tiles) {
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
// Whether the work is split over all SMs: not where a unit's tiles are few, for which the second launch costs more than it saves.
bool split_wanted(int64_t rows, int64_t tiles) { return rows <= 16 && tiles > 2 * kWarps; }

template <typename QT, int D, int BITS, int NT>
int launch_token(const TokenArgs& ta, int ctas, cudaStream_t s) {
  constexpr int kSmem = Tile<D, BITS>::kSmem;
  auto* kernel = kvq_token_kernel<QT, D, BITS, NT>;
  cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
  if (e == cudaSuccess) e = launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kWarps * 32), kSmem, s, ta);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  if (const int rc = check_launch("kvq_attn"); rc != CTDK_OK || !ta.split) return rc;
  e = launch_pdl(kvq_join_kernel<QT, D, BITS, NT>, dim3(static_cast<unsigned>(ta.a.c.B * ta.a.c.Hk)), dim3(D), 0, s, ta, ctas);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  return check_launch("kvq_attn");
}
template <typename QT>
int launch_any(const TokenArgs& ta, int D, int bits, int nt, int ctas, cudaStream_t s) {
  if (D == 64) {
    if (bits == 4) return nt == 1 ? launch_token<QT, 64, 4, 1>(ta, ctas, s) : launch_token<QT, 64, 4, 2>(ta, ctas, s);
    return nt == 1 ? launch_token<QT, 64, 8, 1>(ta, ctas, s) : launch_token<QT, 64, 8, 2>(ta, ctas, s);
  }
  if (bits == 4) return nt == 1 ? launch_token<QT, 128, 4, 1>(ta, ctas, s) : launch_token<QT, 128, 4, 2>(ta, ctas, s);
  return nt == 1 ? launch_token<QT, 128, 8, 1>(ta, ctas, s) : launch_token<QT, 128, 8, 2>(ta, ctas, s);
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
  CTDK_REQUIRE(T >= 0 && H > 0 && H % cache->Hk == 0, "kvq_attn: heads must be a multiple of kv heads");
  const int64_t rows = T * (H / cache->Hk);
  return rows <= 16 ? kvq::part_bytes(cache->D, rows) : 0;
}

int ctdk_kvq_attn(const ctdk_kvq_cache* cache, const void* q, int dtype, int64_t row_stride, int64_t batch_stride, int64_t T, int H,
                  const int32_t* pos, int64_t pos_all, const int32_t* count, int64_t window, int64_t sinks, float scale, void* out,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = kvq::check_cache(cache, "kvq_attn"); rc != CTDK_OK) return rc;
  CTDK_REQUIRE(dtype == CTDK_DTYPE_F32 || dtype == CTDK_DTYPE_BF16, "kvq_attn: dtype must be CTDK_DTYPE_F32 or CTDK_DTYPE_BF16");
  CTDK_REQUIRE(H > 0 && H % cache->Hk == 0, "kvq_attn: heads must be a multiple of kv heads");
  CTDK_REQUIRE(window >= 0 && sinks >= 0, "kvq_attn: window and sinks must not be negative");
  CTDK_REQUIRE(T >= 0 && T <= INT32_MAX / 2 / H, "kvq_attn: bad T");
  CTDK_REQUIRE(pos != nullptr || (pos_all >= 0 && pos_all + T <= cache->capacity), "kvq_attn: positions %lld..%lld exceed the capacity %lld",
               static_cast<long long>(pos_all), static_cast<long long>(pos_all + T), static_cast<long long>(cache->capacity));
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
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  a.status = device_status_word();
  if (a.status == nullptr) return fail(CTDK_ELAUNCH, "kvq_attn: no status word");
  const int64_t rows = T * a.group, units = cache->B * cache->Hk;
  ta.rows = static_cast<int>(rows);
  const int nt = rows <= 8 ? 1 : 2;
  const int64_t tiles = kvq::most_tiles(a, cache->D, cache->bits);
  ta.split = kvq::split_wanted(rows, tiles) ? 1 : 0;
  int64_t ctas = units * ((rows + 8 * nt - 1) / (8 * nt));
  if (ta.split) {
    CTDK_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                     workspace_bytes >= kvq::part_bytes(cache->D, rows),
                 "kvq_attn: the workspace needs %lld bytes, 16-byte aligned", static_cast<long long>(kvq::part_bytes(cache->D, rows)));
    ctas = kvq::split_ctas(cache->D, cache->bits, rows, units, tiles);
  }
  CTDK_REQUIRE(ctas <= INT32_MAX && units <= INT32_MAX, "kvq_attn: too many rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CTDK_DTYPE_F32 ? kvq::launch_any<float>(ta, cache->D, cache->bits, nt, static_cast<int>(ctas), s)
                                 : kvq::launch_any<__nv_bfloat16>(ta, cache->D, cache->bits, nt, static_cast<int>(ctas), s);
}

}  // extern "C"
