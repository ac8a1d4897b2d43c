// Attention of prompts and longer drafts over a key/value cache of 4 or 8 bits, on the tcgen05 tensor cores.
//
// An item is 128 query rows of one key/value head (its query heads side by side, row = token * heads + head) and a range of tiles of
// 128 positions. Persistent CTAs, one per SM, walk the items, longest first. 20 warps:
//   warp 0       TMA producer: codes and scales of keys and of values, two stages of each.
//   warp 1       MMA issuer: S(j) = Q K(j)^T into one of two 128-column buffers in tensor memory, Q from tensor memory;
//                O += P(j) V(j) with P from tensor memory, over S. S(j + 2) is queued right behind P V(j).
//   warps 4-11   softmax, two threads a row, half of the columns each (one thread a row took twice as long as the products): load Q
//                and put it into tensor memory; maxima, exponentials and sums in fp32, in the log2 domain; O is rescaled only when a
//                row's maximum grew by more than 2^8.
//   warps 12-19  turn codes into fp16 tiles, 128-byte-swizzled rows that serve as the K-major keys (four of them) and the MN-major
//                values (the others) alike.
//   warp 2       looks a tile's scales over, a tile ahead of those: exponents, NaN. (Warp 3 only fills a warpgroup.)
// The products take fp16 operands. c * s is not exact in fp16 for every scale s, but c * s * 2^-e is, for the power of two that
// brings a tile's largest scale near the top of the range, unless a scale is far smaller than that one (Span below). Keys have
// an e of their own in every tile (it joins the scores' factor), values one that O is rescaled for when a tile exceeds it. That one is
// shared by the item's rows, whichever of them see the largest values; where an item's scales lie too far apart for it, warp 2 marks the
// item, and its rows are formed once more from the cache in fp32 (exact_rows). fp32 queries
// enter as two fp16 terms (22 bits), and so do the probabilities of fp32 outputs; those of bfloat16 outputs as one.
// With A from tensor memory the products read 64 bytes a clock of shared memory; with both operands there they would wait for it.
// Every mbarrier wait is bounded.
// Measured (B200): 2048 fp32 rows of 16 heads of 128 after 6144 positions in 4 bits (120 GFLOP, executed as two products each): 320 us, 376 TFLOP/s
// of the 1635 that a bfloat16 product reaches, 214 us in bfloat16; 4095 bfloat16 rows of 32 heads of 64 with a window of 512: 110 us. The
// tensor pipe is active in 43 % of the cycles, a scheduler has five warps and issues in 52 %; of the cycles between two issues of a warp,
// loads (of tensor memory, first of all) take 3.6, fixed latencies 1.1, barriers 0.9, missing instructions 0.8. A tile is bound by the softmax threads (two terms a probability: 17 cycles an element and thread) and the
// conversion beside them, which share the instruction cache: code that was unrolled further ran slower (461 -> 297 us when the roles'
// loops were made small). The fp32 softmax spills 72 (128 columns) or 92 bytes.
#include <climits>

#include "kv_quant_attn.h"

namespace ctdk {
namespace kvq {
namespace {

constexpr int TQ = 128, KT = 128;
constexpr int kChunk = 128 * 128;        // bytes of a {64 columns x 128 rows} tile
constexpr float kSlack = 8.0f;
// Probabilities (2^kSlack at most) are held times 2^kLift, sums alike: fp16's smallest step is then 2^-31 of the largest one.
constexpr float kLift = 7.0f;
constexpr int kSoft = 4, kMake = 12;     // first warps of the roles: whole warpgroups, which share out the registers anew
constexpr int kThreads = 20 * 32;
// Registers a thread: 96 at launch, shared out as 64 + 2 * 128 + 2 * 80 = 5 * 96.
constexpr int kRegsLead = 64, kRegsSoft = 128, kRegsMake = 80;
static_assert(kRegsLead + 2 * kRegsSoft + 2 * kRegsMake == 5 * 96, "an increase waits for what the others give back");
// fp32 outputs: the tensor cores cut sums off rather than round them, which over a long row cost 1e-5. O is summed there over this
// many tiles, and the sums of those are added in fp32, in memory that stays in L2 (registers and tensor memory are full).
constexpr int kTogether = 4;
// Tiles whose exponents and NaN marks are kept. Five at least: warp 2 looks keys over up to four tiles ahead of the softmax that reads
// their factor (the keys' stages go by S alone), values up to three (theirs go by P V, which waits for the softmax).
constexpr int kRing = 8;
constexpr int kRoom = 6;                 // powers of two by which values may grow before O is rescaled

// Powers of two that a tile's scales of keys, an item's of values, may lie apart. All products of codes and scales are exact as long as
// the smallest scale does not come below 2^-21 (4 bits: four significant bits, and fp16 has multiples of 2^-24) or 2^-24; that is enough
// for bfloat16 outputs. The tensor cores, though, align products by the exponents that operands are held with, 2^-14 for all subnormal
// ones, and cut off some 26 bits below (seen in their results: 17 bits were left of a value of 2^-23): for fp32 outputs, 22 bits are
// left down to 2^-18. Values may start kRoom lower.
template <typename QT, int BITS>
struct Span {
  static constexpr int kTop = BITS == 4 ? 11 : 7;                    // the largest scale comes to [2^kTop, 2^(kTop + 1))
  static constexpr int kK = kTop + (sizeof(QT) == 4 ? 18 : BITS == 4 ? 21 : 24), kV = kK - kRoom;
};

template <int D, int BITS>
struct Cfg {
  static constexpr int kRow = D * BITS / 8, kGroups = D / kGroup, kChunks = D / 64;
  static constexpr int kCodes = KT * kRow, kScales = KT * kGroups * 2;
  static constexpr int kTile = kChunks * kChunk;                     // a converted tile
  static constexpr int kSmem = 1024 + 4 * kTile + 4 * kCodes + 4 * kScales;
};

struct TcArgs {
  AttnArgs a;
  int rows, row_tiles, splits, items;    // T * group; of 128; ranges of an item's tiles; in all
  uint32_t x64;                          // 0x64006400: fp16 1024
  float* total;                          // fp32: gathered sums, [CTA][TQ * D]
  int* wide;                             // [items] whether an item's scales lie too far apart
};
struct Item {
  int b, h, r0, rows, ks, k0, k1;        // tiles k0 .. k1 - 1 of the visit
  int64_t pos, count;
  Visit v;
};
__device__ __forceinline__ Item item_at(const TcArgs& ta, int it, int splits) {
  const AttnArgs& a = ta.a;
  Item w;
  const int ks = it % splits, i = it / splits, units = a.c.B * a.c.Hk, u = i % units, rt = ta.row_tiles - 1 - i / units;
  w.ks = ks;
  w.b = u / a.c.Hk;
  w.h = u - w.b * a.c.Hk;
  w.r0 = rt * TQ;
  w.rows = min(TQ, ta.rows - w.r0);
  w.pos = a.pos != nullptr ? static_cast<int64_t>(a.pos[w.b]) : a.pos_all;
  w.count = a.count != nullptr ? min(static_cast<int64_t>(a.count[w.b]), static_cast<int64_t>(a.T)) : a.T;
  const int t0 = w.r0 / a.group, t1 = (w.r0 + w.rows - 1) / a.group;
  w.v = visit_of(w.pos, w.count, t0, t1 - t0 + 1, a.c.capacity, a.window, a.sinks, KT);
  w.k0 = static_cast<int>(static_cast<int64_t>(w.v.tiles) * ks / splits);
  w.k1 = static_cast<int>(static_cast<int64_t>(w.v.tiles) * (ks + 1) / splits);
  return w;
}
__device__ __forceinline__ Item item_at(const TcArgs& ta, int it) { return item_at(ta, it, ta.splits); }

__device__ __forceinline__ uint32_t idesc_f16(bool b_mn, int n) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(TQ >> 4) << 24);
}
// The lowest n bits (n below 0: none; from 32 on: all).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(max(-126, min(127, e)) + 127) << 23); }
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}

// Rows r0 .. end - 1 of an item, by one warp, N at a time, from the codes and scales in the cache, in fp32 throughout: a lane a position
// for the scores, a lane D / 32 columns for the output. For items whose scales no single power of two brings into fp16's range: right
// for every scale, and slow (2048 fp32 rows of 16 heads of 128 after 6144 positions, all of them: 29 ms).
template <typename QT, int D, int BITS, int N>
__device__ __forceinline__ void exact_rows(const TcArgs& ta, const Item& w, int r0, int end, int lane) {
  using C = Cfg<D, BITS>;
  constexpr int kOwn = D / 32, kBias = 1 << (BITS - 1), kMask = (1 << BITS) - 1, kWords = kGroup * BITS / 32, kAtOnce = 8;
  const AttnArgs& a = ta.a;
  const int64_t base = (static_cast<int64_t>(w.b) * a.c.Hk + w.h) * a.c.capacity;
  const int col = lane * kOwn;
  auto scale_of = [](uint32_t bits) { return is_nan_scale(bits) ? __int_as_float(0x7fc00000) : __uint_as_float(bits << 16); };
  const unsigned short* k_scales = reinterpret_cast<const unsigned short*>(a.c.scales[0]);
  const unsigned short* v_scales = reinterpret_cast<const unsigned short*>(a.c.scales[1]);
#pragma unroll 1
  for (; r0 < end; r0 += N) {
    const QT* q[N];
    int at[N], last = -1;
    float m[N], l[N], o[N][kOwn];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = w.r0 + min(r0 + n, end - 1), t = r / a.group, hg = r - t * a.group;   // (rows past the end: the last one again)
      at[n] = row_position(w.pos, w.count, t, a.c.capacity);
      last = max(last, at[n]);
      q[n] = static_cast<const QT*>(a.q) + w.b * a.batch_stride + static_cast<int64_t>(t) * a.row_stride + static_cast<int64_t>(w.h * a.group + hg) * D;
      m[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int c = 0; c < kOwn; ++c) o[n][c] = 0.0f;
    }
#pragma unroll 1
    for (int k = 4 * w.k0; k < 4 * w.k1; ++k) {
      const int j0 = w.v.tile_at(k >> 2) * KT + 32 * (k & 3), j = j0 + lane;
      if (j0 > last) continue;
      bool mine = false;
#pragma unroll
      for (int n = 0; n < N; ++n) mine |= sees(at[n], j, a.window, a.sinks);   // (what a row sees lies in the cache)
      const uint32_t seen = __ballot_sync(0xffffffffu, mine);
      if (seen == 0) continue;
      float x[N];
#pragma unroll
      for (int n = 0; n < N; ++n) x[n] = 0.0f;
      if (mine) {
        const uint4* codes = reinterpret_cast<const uint4*>(a.c.codes[0] + (base + j) * C::kRow);
#pragma unroll 1
        for (int g = 0; g < C::kGroups; ++g) {
          const float s = scale_of(k_scales[(base + j) * C::kGroups + g]);
          uint32_t word[kWords];
#pragma unroll
          for (int i = 0; i < kWords / 4; ++i) {
            const uint4 c = codes[g * (kWords / 4) + i];
            word[4 * i] = c.x, word[4 * i + 1] = c.y, word[4 * i + 2] = c.z, word[4 * i + 3] = c.w;
          }
          float sum[N];
#pragma unroll
          for (int n = 0; n < N; ++n) sum[n] = 0.0f;
#pragma unroll
          for (int i = 0; i < kGroup; i += 8) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c)
              v[c] = static_cast<float>(static_cast<int>(word[(i + c) * BITS / 32] >> ((i + c) * BITS % 32) & kMask) - kBias) * s;
#pragma unroll
            for (int n = 0; n < N; ++n) {
              float y[8];
              load8(q[n] + g * kGroup + i, y);
#pragma unroll
              for (int c = 0; c < 8; ++c) sum[n] = fmaf(y[c], v[c], sum[n]);
            }
          }
#pragma unroll
          for (int n = 0; n < N; ++n) x[n] += sum[n];
        }
      }
      float p[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const bool sees_it = mine && sees(at[n], j, a.window, a.sinks);
        const float z = sees_it ? __fmul_rn(x[n], a.scale_log2) : -INFINITY, most = warp_max(z);
        if (most > m[n]) {
          const float f = ex2(m[n] - most);
          m[n] = most;
          l[n] *= f;
#pragma unroll
          for (int c = 0; c < kOwn; ++c) o[n][c] *= f;
        }
        p[n] = sees_it ? ex2(z - (m[n] == -INFINITY ? 0.0f : m[n])) : 0.0f;
        l[n] += warp_sum(p[n]);
      }
      float sum[N][kOwn];
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int c = 0; c < kOwn; ++c) sum[n][c] = 0.0f;
#pragma unroll 1
      for (int i0 = 0; i0 < 32; i0 += kAtOnce) {
        float v[kAtOnce][kOwn];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const bool there = (seen >> (i0 + i) & 1u) != 0;
          const int64_t row = base + j0 + (there ? i0 + i : __ffs(seen) - 1);
          const float s = scale_of(v_scales[row * C::kGroups + col / kGroup]);
#pragma unroll
          for (int c = 0; c < kOwn; ++c)
            v[i][c] = static_cast<float>(static_cast<int>(a.c.codes[1][row * C::kRow + (col + c) * BITS / 8] >> ((col + c) * BITS % 8) & kMask) - kBias) * s;
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int n = 0; n < N; ++n) {
            // (a value that the row does not see may be NaN: it is no part of the sum)
            const float pi = __shfl_sync(0xffffffffu, p[n], i0 + i);
            const bool sees_it = sees(at[n], j0 + i0 + i, a.window, a.sinks);
#pragma unroll
            for (int c = 0; c < kOwn; ++c) sum[n][c] = sees_it ? fmaf(pi, v[i][c], sum[n][c]) : sum[n][c];
          }
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int c = 0; c < kOwn; ++c) o[n][c] += sum[n][c];
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (r0 + n < end) {
        const int r = w.r0 + r0 + n, t = r / a.group, hg = r - t * a.group;
        QT* dst = static_cast<QT*>(a.out) + ((static_cast<int64_t>(w.b) * a.T + t) * a.H + w.h * a.group + hg) * D + col;
#pragma unroll
        for (int c = 0; c < kOwn; ++c) store_out(dst + c, at[n] >= 0 ? o[n][c] / l[n] : 0.0f);
      }
  }
}

// The marked items of a call without ranges (the join sees to those of a call with ranges): the CTA's own, behind its loop over them, by
// its softmax warps. A call, not in line, and for fp32 queries over 128 columns a launch of its own: registers that the softmax loses to it
// cost more there (2048 rows after 6144 positions 330 us, in line 380; a launch 3 us on top of 315. The others: the call 0 to 1 us, a launch 3).
template <typename QT, int D>
constexpr bool kOwnLaunch = sizeof(QT) == 4 && D == 128;
template <typename QT, int D, int BITS, int N>
__device__ __forceinline__ void exact_items(const TcArgs& ta, int warp) {
  for (int it = blockIdx.x; it < ta.items; it += gridDim.x)
    if (ta.wide[it] != 0) {
      const Item w = item_at(ta, it);
      exact_rows<QT, D, BITS, N>(ta, w, warp * 16, min(warp * 16 + 16, w.rows), threadIdx.x & 31);
    }
}
template <typename QT, int D, int BITS>
__device__ __noinline__ void exact_call(const TcArgs* ta) {
  exact_items<QT, D, BITS, 2>(*ta, static_cast<int>(threadIdx.x >> 5) - kSoft);
}
template <typename QT, int D, int BITS>
__global__ void __launch_bounds__(256) kvq_prompt_exact_kernel(const TcArgs ta) {
  pdl_launch();
  pdl_wait();
  exact_items<QT, D, BITS, 4>(ta, threadIdx.x >> 5);
}

template <typename QT, int D, int BITS>
__global__ void __launch_bounds__(kThreads, 1) kvq_prompt_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                                                                   const __grid_constant__ TcArgs ta) {
  using C = Cfg<D, BITS>;
  constexpr int NT = sizeof(QT) == 4 ? 2 : 1;          // fp16 terms of a query, of a probability
  constexpr uint32_t kColS = 0, kColO = 2 * KT, kColQ = 2 * KT + 128;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bars[27 + kRing];
  __shared__ uint32_t tmem_slot;
  __shared__ float row_x[2][2][TQ];                    // what the two threads of a row tell each other, by parity of the exchange
  __shared__ int exp_k[kRing], exp_v[kRing];           // exponents of a tile's keys and values
  __shared__ float scale_k[kRing], shrink_o[kRing];    // 2^exp_k; what O has to be multiplied by, as exp_v has moved
  __shared__ uint32_t nan_any[kRing];
  __shared__ int any_wide;                             // of this CTA's items
  __shared__ uint8_t nan_of[kRing][KT];                // groups of values that are NaN, by position
  const AttnArgs& a = ta.a;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* k_s = smem;                           // [2] converted tiles
  unsigned char* v_s = k_s + 2 * C::kTile;
  unsigned char* codes_s = v_s + 2 * C::kTile;         // [2][keys, values]
  unsigned char* scales_s = codes_s + 4 * C::kCodes;   // [2][keys, values]
  uint64_t* in_full = bars;          // [2][keys, values]: codes and scales are there
  uint64_t* in_empty = bars + 4;     // [2][keys, values]: converted
  uint64_t* k_full = bars + 8;       // [2] converted keys
  uint64_t* k_empty = bars + 10;
  uint64_t* v_full = bars + 12;
  uint64_t* v_empty = bars + 14;
  uint64_t* s_full = bars + 16;      // [2] S(g) is in tensor memory
  uint64_t* p_ready = bars + 18;     // [2] P(g) has replaced S(g)
  uint64_t* q_ready = bars + 20;     // Q of the item is in tensor memory, O of the one before has been read
  uint64_t* pv_full = bars + 21;     // O += P(g) V(g) has finished (one phase per step)
  uint64_t* o_full = bars + 22;      // the item's last one has
  uint64_t* looked = bars + 23;      // [2][keys, values]: the scales have been looked over, for the warps that convert
  uint64_t* told = bars + 27;        // [kRing] the same of values, for the MMA issuer and the softmax behind it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 27 + kRing; ++i) mbar_init(&bars[i], (i >= 4 && i < 10) || i == 12 || i == 13 ? 4 : i >= 18 && i < 21 ? 256 : 1);
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  pdl_wait();
  // g = running count of tiles over all items of this CTA: stage g & 1, phase (g >> 1) & 1
  if (warp < kSoft) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLead));
  if (warp == 0) {
    uint32_t g = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < ta.items && ok; it += gridDim.x) {
      const Item w = item_at(ta, it);
      const int bh = w.b * a.c.Hk + w.h;
      for (int k = w.k0; k < w.k1 && ok; ++k, ++g) {
        const int st = g & 1u, j = w.v.tile_at(k) * KT;
        const int there = static_cast<int>(min(static_cast<int64_t>(KT), a.c.capacity - j));   // positions that the cache has
        const int64_t sc = (static_cast<int64_t>(bh) * a.c.capacity + j) * C::kGroups;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ok = ok && wait_w(&in_empty[2 * st + i], ((g >> 1) & 1u) ^ 1u, a.status, 220 + i);
          if (ok && lane == 0) {
            uint64_t* bar = &in_full[2 * st + i];
            mbar_expect_tx(bar, C::kCodes + there * C::kGroups * 2);
            tma_load_3d(codes_s + (2 * st + i) * C::kCodes, i ? &tm_v : &tm_k, bar, 0, j, bh);
            bulk_load(scales_s + (2 * st + i) * C::kScales, a.c.scales[i] + sc, there * C::kGroups * 2, bar);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 1) {
    // The whole warp runs this role converged; one elected lane issues each MMA / commit.
    const uint32_t idesc_s = idesc_f16(false, KT), idesc_pv = idesc_f16(true, D);
    const uint32_t k_base = smem_u32(k_s), v_base = smem_u32(v_s);
    uint32_t g0 = 0, n_it = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < ta.items && ok; it += gridDim.x) {
      const Item w = item_at(ta, it);
      const int steps = w.k1 - w.k0;
      if (steps <= 0) continue;
      auto issue_s = [&](int j) {
        const uint32_t g = g0 + static_cast<uint32_t>(j), s = g & 1u;
        if (!wait_w(&k_full[s], (g >> 1) & 1u, a.status, 222) || !wait_w(&told[g % kRing], (g / kRing) & 1u, a.status, 233)) return false;
        tc_fence_after();
        const uint64_t kd = make_smem_desc(k_base + s * C::kTile, 16, 1024, kLayoutSw128);
        const uint32_t ts = tmem_base + kColS + s * KT, tq = tmem_base + kColQ;
#pragma unroll
        for (int x = NT - 1; x >= 0; --x)              // the small terms first: sums are cut off at their own size
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            umma_bf16_ta_w(ts, tq + static_cast<uint32_t>(x * (D / 2) + ks * 8), kd + (((ks >> 2) * kChunk + (ks & 3) * 32) >> 4), idesc_s,
                           x != NT - 1 || ks != 0 ? 1u : 0u);
        umma_commit_w(&k_empty[s]);
        umma_commit_w(&s_full[s]);
        return true;
      };
      if (!wait_w(q_ready, n_it & 1u, a.status, 223)) break;
      ++n_it;
      tc_fence_after();
      ok = issue_s(0);
      if (ok && steps > 1) ok = issue_s(1);
      for (int j = 0; j < steps && ok; ++j) {
        const uint32_t g = g0 + static_cast<uint32_t>(j), s = g & 1u, ph = (g >> 1) & 1u;
        ok = wait_w(&v_full[s], ph, a.status, 224) && wait_w(&p_ready[s], ph, a.status, 225);
        if (!ok) break;
        tc_fence_after();
        // B: 16 key rows (two 8-row swizzle groups, SBO) of every 64-column chunk of V (LBO)
        const uint64_t vd = make_smem_desc(v_base + s * C::kTile, kChunk, 1024, kLayoutSw128);
        const uint32_t ts = tmem_base + kColS + s * KT;
#pragma unroll
        for (int x = NT - 1; x >= 0; --x)
#pragma unroll
          for (int kb = 0; kb < KT / 16; ++kb)
            umma_bf16_ta_w(tmem_base + kColO, ts + static_cast<uint32_t>((kb >> 1) * 32 + x * 16 + (kb & 1) * 8), vd + ((kb * 2048) >> 4), idesc_pv,
                           x != NT - 1 || kb != 0 || (NT == 2 ? j % kTogether != 0 : j != 0) ? 1u : 0u);
        umma_commit_w(&v_empty[s]);
        umma_commit_w(pv_full);
        if (j == steps - 1) umma_commit_w(o_full);
        if (j + 2 < steps) ok = issue_s(j + 2);
      }
      g0 += static_cast<uint32_t>(steps);
    }
    __syncwarp();
  } else if (warp == 2) {
    // Exponents of a tile's keys and values, and which groups of its values are NaN. What none of the rows sees must not matter.
    uint32_t g = 0;
    bool ok = true, marked = false;
    for (int it = blockIdx.x; it < ta.items && ok; it += gridDim.x) {
      const Item w = item_at(ta, it);
      int vref = 0, vtop = -1, vlow = 0x7fff;          // (exponents of scales as their bits have them)
      bool wide = false;
      for (int k = w.k0; k < w.k1 && ok; ++k, ++g) {
        const uint32_t st = g & 1u, ph = (g >> 1) & 1u;
        const int j0 = w.v.tile_at(k) * KT;
#pragma unroll 1
        for (int which = 0; which < 2 && ok; ++which) {
          ok = wait_w(&in_full[2 * st + which], ph, a.status, 243);
          if (!ok) break;
          const unsigned char* p = scales_s + (2 * st + which) * C::kScales;
          // The largest scale and the smallest one that is not zero (less one, so that zero becomes the largest), two a word.
          auto words = [&](int row, uint32_t (&sw)[C::kGroups / 2]) {
            if constexpr (C::kGroups == 4) {
              const uint2 x = *reinterpret_cast<const uint2*>(p + row * 8);
              sw[0] = x.x, sw[C::kGroups / 2 - 1] = x.y;
            } else {
              sw[0] = *reinterpret_cast<const uint32_t*>(p + row * 4);
            }
            const int at = j0 + row;
            return at < w.v.hi_row && (at >= w.v.lo_row || a.window == 0 || w.v.lo_row - at < a.window || at < a.sinks);
          };
          uint32_t most = 0, least = 0xffffffffu, any = 0;
#pragma unroll
          for (int i = 0; i < KT / 32; ++i) {
            uint32_t sw[C::kGroups / 2];
            const bool seen = words(32 * i + lane, sw);
#pragma unroll
            for (int y = 0; y < C::kGroups / 2; ++y) {
              most = __vmaxu2(most, seen ? sw[y] & 0x7fff7fffu : 0u);
              least = __vminu2(least, seen ? ((sw[y] | 0x80008000u) - 0x00010001u) ^ 0x80008000u : 0xffffffffu);
            }
          }
          uint32_t big = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
          if (is_nan_scale(big)) {                     // the largest of the others, and where the NaN are
            big = 0;
#pragma unroll 1
            for (int i = 0; i < KT / 32; ++i) {
              uint32_t sw[C::kGroups / 2], nan = 0;
              const bool seen = words(32 * i + lane, sw);
#pragma unroll
              for (int y = 0; y < C::kGroups; ++y) {
                const uint32_t b = (y & 1 ? sw[y / 2] >> 16 : sw[y / 2]) & 0x7fffu;
                if (is_nan_scale(b)) nan |= 1u << y;
                else if (seen) big = max(big, b);
              }
              if (!seen) nan = 0;
              any |= nan;
              if (which == 1) nan_of[g % kRing][32 * i + lane] = static_cast<uint8_t>(nan);
            }
            big = __reduce_max_sync(0xffffffffu, big);
            any = __any_sync(0xffffffffu, any != 0) ? 1u : 0u;
          }
          const int e = big == 0 ? (which ? -120 : 0) : max(static_cast<int>(big >> 7) - 127 - Span<QT, BITS>::kTop, -120);
          if (which == 0) {
            exp_k[g % kRing] = e;                      // (all lanes: the same)
            scale_k[g % kRing] = pow2(e);
          } else {
            int moved = 0;
            if (k == w.k0) {
              vref = e + kRoom;
            } else if (e > vref) {
              moved = e + kRoom - vref;
              vref += moved;
            }
            exp_v[g % kRing] = vref;
            shrink_o[g % kRing] = pow2(-moved);
            nan_any[g % kRing] = any;
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&looked[2 * st + which]);
            if (which == 1) mbar_arrive(&told[g % kRing]);
          }
          if (big != 0) {                              // (behind what others wait for)
            const int top = static_cast<int>(big >> 7), bottom = static_cast<int>((__reduce_min_sync(0xffffffffu, min(least & 0xffffu, least >> 16)) + 1u) >> 7);
            if (which == 0) wide |= top - bottom > Span<QT, BITS>::kK;
            else vtop = max(vtop, top), vlow = min(vlow, bottom);
          }
        }
      }
      wide |= vtop - vlow > Span<QT, BITS>::kV;
      marked |= wide;
      if (lane == 0) ta.wide[it] = wide ? 1 : 0;
    }
    if constexpr (!kOwnLaunch<QT, D>) {
      if (lane == 0) any_wide = ok && marked && ta.splits == 1 ? 1 : 0;
      __syncwarp();
      asm volatile("barrier.cta.arrive 5, 288;" ::: "memory");   // with the softmax warps
    }
  }
  } else if (warp < kMake) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
    const int quarter = warp & 3, half = (warp - kSoft) >> 2;   // tensor-memory lanes of this warp; of the columns, 64 half ..
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t to = tmem_base + kColO + lane_off + half * (D / 2), tq = tmem_base + kColQ + lane_off;
    const int rr = quarter * 32 + lane;
    uint32_t g0 = 0, n_done = 0, n_ex = 0;
    bool ok = true;
    // Adds the thread's part of O, times `now`, to what it has gathered, times `then` (nothing yet: any is false).
    float4* total = reinterpret_cast<float4*>(ta.total) + static_cast<int64_t>(blockIdx.x) * (TQ * D / 4) + (threadIdx.x - kSoft * 32);
    auto gather = [&](bool any, float now, float then) {
#pragma unroll 1
      for (int p = 0; p < D / 64; ++p) {
        float4 t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = any ? total[(8 * p + i) * 256] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float o[32];
        tmem_ld_32x32(to + p * 32, o);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          total[(8 * p + i) * 256] = make_float4(fmaf(t[i].x, then, o[4 * i] * now), fmaf(t[i].y, then, o[4 * i + 1] * now),
                                                 fmaf(t[i].z, then, o[4 * i + 2] * now), fmaf(t[i].w, then, o[4 * i + 3] * now));
      }
    };
    // The other thread's value of the row. The two warps also agree on `ok`: they give up together.
    auto other = [&](float mine) {
      float* x = &row_x[n_ex & 1u][0][0];
      ++n_ex;
      x[half * TQ + rr] = mine;
      int all_ok;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, 64, p;\n selp.b32 %0, 1, 0, q;\n}"
                   : "=r"(all_ok) : "r"(static_cast<int>(ok)), "r"(1 + quarter) : "memory");
      ok = all_ok != 0;
      return x[(half ^ 1) * TQ + rr];
    };
    for (int it = blockIdx.x; it < ta.items && ok; it += gridDim.x) {
      const Item w = item_at(ta, it);
      const int steps = w.k1 - w.k0, r = w.r0 + rr, t = r / a.group, hg = r - t * a.group;
      const bool live = rr < w.rows;
      const int at = live ? row_position(w.pos, w.count, t, a.c.capacity) : -1;
      float m_ref = -INFINITY, l = 0.0f, o_scale = 0.0f;
      float pending = 1.0f, before = 1.0f;             // what the gathered sums, O itself, have to be multiplied by
      uint32_t poison = 0;                             // groups of columns that have met a NaN
      if (steps > 0) {
        // Q: a power of two brings the row's largest value near 64; terms into tensor memory, in the order of the converted keys
        const QT* src = static_cast<const QT*>(a.q) + w.b * a.batch_stride + static_cast<int64_t>(t) * a.row_stride +
                        static_cast<int64_t>(w.h * a.group + hg) * D + half * (D / 2);
        float big = 0.0f;
        if (live)
#pragma unroll 4
          for (int i = 0; i < D / 2; i += 8) {
            float x[8];
            load8(src + i, x);
#pragma unroll
            for (int c = 0; c < 8; ++c) big = fmaxf(big, fabsf(x[c]));
          }
        big = fmaxf(big, other(big));
        const int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;              // 128: not finite
        const int up = big == 0.0f || e == 128 ? 0 : min(6 - e, 126);
        const float f = a.scale_log2 < 0.0f ? -pow2(up) : pow2(up);
        const float factor = fabsf(a.scale_log2) * pow2(-up);   // 2^-126 to 2^121
#pragma unroll 1
        for (int i = 0; i < D / 2; i += 32) {
          uint32_t q16[NT][16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x[8] = {};
            if (live) load8(src + i + 8 * k, x);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // 4 bits: a word's codes come as pairs (c, c + 4); 8 bits: in order
              float u = (BITS == 4 ? x[c] : x[2 * c]) * f, v = (BITS == 4 ? x[c + 4] : x[2 * c + 1]) * f;
#pragma unroll
              for (int y = 0; y < NT; ++y) {
                q16[y][4 * k + c] = pack_f16(u, v);
                if (y + 1 < NT) {
                  float a0, a1;
                  unpack_f16(q16[y][4 * k + c], a0, a1);
                  u -= a0, v -= a1;
                }
              }
            }
          }
#pragma unroll
          for (int y = 0; y < NT; ++y) tmem_st_32x16(tq + static_cast<uint32_t>(y * (D / 2) + half * (D / 4) + i / 2), q16[y]);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(q_ready);
        // 64 positions from j0 on are seen by every row: j0 from plain_lo to plain_hi, or up to plain_sink
        const int plain_lo = a.window == 0 ? 0 : w.v.hi_row - a.window, plain_hi = w.v.lo_row - 63;
        const int plain_sink = a.window == 0 ? -1 : min(a.sinks - 64, plain_hi);
        for (int j = 0; j < steps; ++j) {
          const uint32_t g = g0 + static_cast<uint32_t>(j), s = g & 1u;
          const int j0 = w.v.tile_at(w.k0 + j) * KT + 64 * half;
          const bool plain = (j0 >= plain_lo && j0 <= plain_hi) || j0 <= plain_sink;
          const uint32_t ts = tmem_base + kColS + s * KT + lane_off + 64 * half;
          ok = ok && wait_w(&s_full[s], (g >> 1) & 1u, a.status, 230);
          tc_fence_after();
          if (quarter * 32 >= w.rows) {                // none of the warp's rows is there: whatever lies in theirs may stay
            mbar_arrive(&p_ready[s]);
            continue;
          }
          float x[64];
          tmem_ld_32x64_nowait(ts, x);
          float sc = fminf(fmaxf(factor * scale_k[g % kRing], 0x1p-126f), 0x1p127f);   // (finite: scores of zero stay)
          const float shrink = shrink_o[g % kRing];
          tmem_wait_ld();
          if (!plain) {
            // which of 32 positions the row sees, as bits: up to its own, from the window's first on or below the sinks
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int base = j0 + 32 * q;
              const uint32_t from = a.window == 0 ? 0xffffffffu : ~below(at - a.window + 1 - base) | below(a.sinks - base);
              const uint32_t bits = below(at + 1 - base) & from;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if ((bits >> i & 1u) == 0) x[32 * q + i] = -INFINITY;
            }
          }
          float mx;
          {
            float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
            for (int i = 4; i + 7 < 64; i += 8) {
              m0 = fmax3(m0, x[i], x[i + 1]);
              m1 = fmax3(m1, x[i + 2], x[i + 3]);
              m2 = fmax3(m2, x[i + 4], x[i + 5]);
              m3 = fmax3(m3, x[i + 6], x[i + 7]);
            }
            mx = __fmul_rn(fmax3(fmax3(m0, x[60], x[61]), fmax3(m1, x[62], x[63]), fmaxf(m2, m3)), sc);
          }
          // What the reference point was rounded by, the difference below takes into the exponent, for all positions alike; from 2^23
          // on that could leave fp16's range, and the scores are rounded first.
          if (__builtin_expect(fabsf(mx) > 0x1p23f && mx != -INFINITY, 0)) {
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] = __fmul_rn(x[i], sc);
            sc = 1.0f;
          }
          // Most tiles move no reference point: one barrier tells the two warps of these rows so.
          int move;
          asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 64, p;\n selp.b32 %0, 1, 0, q;\n}"
                       : "=r"(move) : "r"(static_cast<int>(mx - m_ref > kSlack || shrink != 1.0f || !ok)), "r"(1 + quarter) : "memory");
          if (move != 0) {
            const float most = fmaxf(mx, other(mx));
            if (!ok) break;
            float c = 1.0f;
            if (most - m_ref > kSlack) {
              c = ex2(m_ref - most);
              m_ref = most;
            }
            pending *= c * shrink;
            if (j != 0 && (NT == 1 || j % kTogether != 0)) {
              // P V(g-1) must have landed before the accumulator is touched; P V(g) cannot start before every
              // row has arrived at p_ready below. Each thread of a row rescales half of the columns.
              ok = wait_w(pv_full, (g - 1u) & 1u, a.status, 231);
              tc_fence_after();
              const float co = c * shrink;
#pragma unroll 1
              for (int p = 0; p < D / 64; ++p) {
                float o[32];
                tmem_ld_32x32(to + p * 32, o);
#pragma unroll
                for (int i = 0; i < 32; i += 2) fmul2(o[i], o[i + 1], o[i], o[i + 1], co, co);
                tmem_st_32x32(to + p * 32, *reinterpret_cast<uint32_t(*)[32]>(o));
                tmem_wait_st();
              }
            }
            l *= c;
            before = c * shrink;
          }
          if constexpr (NT == 2) {
            if (j != 0 && j % kTogether == 0) {        // the sums of the tiles before join the rest
              ok = ok && wait_w(pv_full, (g - 1u) & 1u, a.status, 234);
              tc_fence_after();
              gather(j != kTogether, before, pending);
              pending = 1.0f;
            }
            before = 1.0f;
          }
          const float neg_m = (m_ref == -INFINITY ? 0.0f : -m_ref) + kLift;
          float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
          for (int q = 0; q < 2; ++q) {                // 32 columns of scores make room for 16 of each term
            uint32_t p16[NT][16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              // (packed pairs of fp32 measured slower here: 20 cycles an element of two terms against 17)
              const float u = ex2(fmaf(x[32 * q + i], sc, neg_m)), v = ex2(fmaf(x[32 * q + i + 1], sc, neg_m));
              s0 += u;
              s1 += v;
              if constexpr (NT == 2) {                 // the upper eleven bits, and the rest
                const float u1 = __uint_as_float(__float_as_uint(u) & 0xffffe000u), v1 = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
                p16[0][i >> 1] = pack_f16(u1, v1);
                p16[NT - 1][i >> 1] = pack_f16(u - u1, v - v1);
              } else {
                p16[0][i >> 1] = pack_f16(u, v);
              }
            }
#pragma unroll
            for (int y = 0; y < NT; ++y) tmem_st_32x16(ts + 32 * q + 16 * y, p16[y]);
          }
          tmem_wait_st();
          tc_fence_before();
          if (nan_any[g % kRing] != 0)                 // NaN values: zeros in the tile; the rows that see them get NaN
#pragma unroll 1
            for (int i = 0; i < 64; ++i)
              if (nan_of[g % kRing][64 * half + i] != 0 && sees(at, j0 + i, a.window, a.sinks)) poison |= nan_of[g % kRing][64 * half + i];
          if (j == steps - 1) o_scale = pow2(exp_v[g % kRing]);
          mbar_arrive(&p_ready[s]);
          l += s0 + s1;
        }
        g0 += static_cast<uint32_t>(steps);
        // The item's last P V. The next item's first one cannot start before these threads have read O and arrived at q_ready.
        ok = ok && wait_w(o_full, n_done & 1u, a.status, 232);
        ++n_done;
        tc_fence_after();
        l += other(l);
        poison |= __float_as_uint(other(__uint_as_float(poison)));
        if (!ok) break;
      }
      float* part = ta.splits > 1 ? a.part + static_cast<int64_t>(it) * TQ * (D + 2) : nullptr;
      const float f = part != nullptr ? o_scale : (at >= 0 ? o_scale / l : 0.0f);
      QT* dst = static_cast<QT*>(a.out) + ((static_cast<int64_t>(w.b) * a.T + t) * a.H + w.h * a.group + hg) * D + half * (D / 2);
#pragma unroll 1
      for (int p = 0; p < D / 64; ++p) {
        float o[32];
        if (steps > 0) {
          tmem_ld_32x32(to + p * 32, o);               // warp-collective: rows past the end take part too
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        }
        if (NT == 2 && steps > kTogether) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 t = total[(8 * p + i) * 256];
            o[4 * i] = fmaf(t.x, pending, o[4 * i]);
            o[4 * i + 1] = fmaf(t.y, pending, o[4 * i + 1]);
            o[4 * i + 2] = fmaf(t.z, pending, o[4 * i + 2]);
            o[4 * i + 3] = fmaf(t.w, pending, o[4 * i + 3]);
          }
        }
        const bool nan = (poison >> (half * (D / 64) + p) & 1u) != 0, none = part == nullptr && at < 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = none ? 0.0f : nan ? __int_as_float(0x7fc00000) : o[i] * f;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          // columns as they came: pairs (c, c + 4) of eight, or in order
          const float y[8] = {o[i], BITS == 4 ? o[i + 2] : o[i + 1], BITS == 4 ? o[i + 4] : o[i + 2], BITS == 4 ? o[i + 6] : o[i + 3],
                              BITS == 4 ? o[i + 1] : o[i + 4], BITS == 4 ? o[i + 3] : o[i + 5], BITS == 4 ? o[i + 5] : o[i + 6], o[i + 7]};
          if (part != nullptr) {
            float* x = part + rr * D + half * (D / 2) + 32 * p + i;
            store4(x, y[0], y[1], y[2], y[3]);
            store4(x + 4, y[4], y[5], y[6], y[7]);
          } else if (live) {
            store4(dst + 32 * p + i, y[0], y[1], y[2], y[3]);
            store4(dst + 32 * p + i + 4, y[4], y[5], y[6], y[7]);
          }
        }
        __syncwarp();
      }
      if (part != nullptr && half == 0) {
        part[TQ * D + rr] = m_ref - kLift;
        part[TQ * D + TQ + rr] = l;
      }
      tc_fence_before();
    }
    if constexpr (!kOwnLaunch<QT, D>) {
      asm volatile("barrier.cta.sync 5, 288;" ::: "memory");
      if (any_wide != 0) exact_call<QT, D, BITS>(&ta);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMake));
    // Four warps convert keys, four values, each at its own pace. A thread has one position of a tile: its swizzles keep the reads
    // and the writes of neighbouring lanes off each other's banks.
    const int which = (warp - kMake) >> 2, row = ((warp - kMake) & 3) * 32 + lane;
    const uint32_t row_at = static_cast<uint32_t>(row * C::kRow), row_swz = (row_at >> 3) & (C::kRow - 16u);   // as TMA has written it
    const uint32_t dst_row = static_cast<uint32_t>(row) * 128u, dst_swz = static_cast<uint32_t>(row & 7) << 4;
    uint64_t *full = which ? v_full : k_full, *empty = which ? v_empty : k_empty;
    uint32_t g = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < ta.items && ok; it += gridDim.x) {
      const Item w = item_at(ta, it);
#pragma unroll 1
      for (int k = w.k0; k < w.k1; ++k, ++g) {
        const uint32_t st = g & 1u, ph = (g >> 1) & 1u;
        const int at = w.v.tile_at(k) * KT + row;
        // (that the scales have been looked over says that the codes are there too)
        ok = wait_w(&looked[2 * st + which], ph, a.status, 240) && wait_w(&empty[st], ph ^ 1u, a.status, 242);
        if (!ok) break;
        const int ex = which ? exp_v[g % kRing] : exp_k[g % kRing];
        const uint32_t src = smem_u32(codes_s) + (2 * st + which) * C::kCodes + row_at;
        const uint32_t dst = smem_u32(which ? v_s : k_s) + st * C::kTile + dst_row;
        const uint32_t scale = smem_u32(scales_s) + (2 * st + which) * C::kScales + static_cast<uint32_t>(row * C::kGroups * 2);
        const bool seen = at < w.v.hi_row && (at >= w.v.lo_row || a.window == 0 || w.v.lo_row - at < a.window || at < a.sinks);
        const float up = seen ? pow2(-ex) : 0.0f;
#pragma unroll 1
        for (int u = 0; u < C::kRow / 16; ++u) {       // 16 bytes: a group of 4-bit codes, half of one of 8-bit codes
          uint32_t wd[4], sb;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(wd[0]), "=r"(wd[1]), "=r"(wd[2]), "=r"(wd[3]) : "r"(src + ((16u * u) ^ row_swz)));
          {
            unsigned short x;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(scale + 2u * (BITS == 4 ? u : u / 2)));
            sb = x;
          }
          float sf = __uint_as_float(sb << 16);
          if (is_nan_scale(sb)) sf = which || !seen ? 0.0f : __int_as_float(0x7fc00000);
          sf *= up;
          const uint32_t su = pack_f16(sf, sf);        // the group's scale under the tile's power of two, twice
          if constexpr (BITS == 4) {
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {           // a word: eight columns
              const uint32_t v = wd[k4] >> 8;
              uint32_t y[4];
              y[0] = add_f16x2((wd[k4] & 0x000f000fu) | ta.x64, 0xe408e408u);               // 1024 + u - 1032
              y[1] = fma_f16x2((wd[k4] & 0x00f000f0u) | ta.x64, 0x2c002c00u, 0xd480d480u);  // (1024 + 16 u) / 16 - 72
              y[2] = add_f16x2((v & 0x000f000fu) | ta.x64, 0xe408e408u);
              y[3] = fma_f16x2((v & 0x00f000f0u) | ta.x64, 0x2c002c00u, 0xd480d480u);
#pragma unroll
              for (int c = 0; c < 4; ++c) y[c] = mul_f16x2(y[c], su);
              sts128(dst + (u >> 1) * kChunk + (dst_swz ^ (16u * ((u & 1) * 4 + k4))), y[0], y[1], y[2], y[3]);
            }
          } else {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {           // two words: eight columns
              uint32_t y[4];
              y[0] = add_f16x2(prmt(wd[2 * k2], ta.x64, 0x5150), 0xe480e480u);              // 1024 + u - 1152
              y[1] = add_f16x2(prmt(wd[2 * k2], ta.x64, 0x5352), 0xe480e480u);
              y[2] = add_f16x2(prmt(wd[2 * k2 + 1], ta.x64, 0x5150), 0xe480e480u);
              y[3] = add_f16x2(prmt(wd[2 * k2 + 1], ta.x64, 0x5352), 0xe480e480u);
#pragma unroll
              for (int c = 0; c < 4; ++c) y[c] = mul_f16x2(y[c], su);
              sts128(dst + (u >> 2) * kChunk + (dst_swz ^ (16u * ((u & 3) * 2 + k2))), y[0], y[1], y[2], y[3]);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[st]);
          mbar_arrive(&in_empty[2 * st + which]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the ranges of the items: a CTA takes 16 rows of one, a thread a column (or two rows' columns). A marked one is formed anew.
template <typename QT, int D, int BITS>
__global__ void __launch_bounds__(256) kvq_prompt_join_kernel(const TcArgs ta) {
  const AttnArgs& a = ta.a;
  pdl_launch();
  pdl_wait();
  const int i = blockIdx.x / (TQ / 16), units = a.c.B * a.c.Hk, u = i % units, rt = ta.row_tiles - 1 - i / units;
  const int b = u / a.c.Hk, h = u - b * a.c.Hk;
  bool wide = false;
  for (int k = 0; k < ta.splits; ++k) wide |= ta.wide[i * ta.splits + k] != 0;
  if (wide) {
    const Item w = item_at(ta, i, 1);
    const int rr = static_cast<int>(blockIdx.x % (TQ / 16)) * 16 + static_cast<int>(threadIdx.x >> 5) * 2;
    exact_rows<QT, D, BITS, 2>(ta, w, rr, min(rr + 2, w.rows), threadIdx.x & 31);
    return;
  }
  const float* part = a.part + static_cast<int64_t>(i) * ta.splits * TQ * (D + 2);
  const int64_t pos = a.pos != nullptr ? static_cast<int64_t>(a.pos[b]) : a.pos_all;
  const int64_t count = a.count != nullptr ? min(static_cast<int64_t>(a.count[b]), static_cast<int64_t>(a.T)) : a.T;
  for (int e = threadIdx.x; e < 16 * D; e += 256) {
    const int rr = static_cast<int>(blockIdx.x % (TQ / 16)) * 16 + e / D, d = e % D, r = rt * TQ + rr;
    if (r >= ta.rows) continue;
    float m = -INFINITY;
#pragma unroll 8
    for (int k = 0; k < ta.splits; ++k) m = fmaxf(m, part[static_cast<int64_t>(k) * TQ * (D + 2) + TQ * D + rr]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, s = 0.0f;
#pragma unroll 8
    for (int k = 0; k < ta.splits; ++k) {
      const float* p = part + static_cast<int64_t>(k) * TQ * (D + 2);
      const float w = ex2(p[TQ * D + rr] - ref);
      l += w * p[TQ * D + TQ + rr];
      s += w * p[rr * D + d];
    }
    const int t = r / a.group, hg = r - t * a.group;
    const float x = row_position(pos, count, t, a.c.capacity) >= 0 ? s / l : 0.0f;
    QT* out = static_cast<QT*>(a.out) + ((static_cast<int64_t>(b) * a.T + t) * a.H + h * a.group + hg) * D + d;
    store_out(out, x);
  }
}

template <typename QT, int D, int BITS>
int launch(const TcArgs& ta, cudaStream_t s) {
  using C = Cfg<D, BITS>;
  CUtensorMap m[2];
  const Cache& c = ta.a.c;
  const uint64_t dims[3] = {C::kRow, static_cast<uint64_t>(c.capacity), static_cast<uint64_t>(c.B) * c.Hk};
  const uint64_t strides[2] = {C::kRow, static_cast<uint64_t>(c.capacity) * C::kRow};
  const uint32_t box[3] = {C::kRow, KT, 1};
  for (int i = 0; i < 2; ++i)
    if (const int rc = encode_tensor_map_u8(&m[i], c.codes[i], 3, dims, strides, box); rc != CTDK_OK) return rc;
  auto* kernel = kvq_prompt_kernel<QT, D, BITS>;
  const int ctas = ta.items < sm_count() ? ta.items : sm_count();
  cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), C::kSmem);
  if (e == cudaSuccess) e = launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), C::kSmem, s, m[0], m[1], ta);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  if (const int rc = check_launch("kvq_attn"); rc != CTDK_OK || (ta.splits == 1 && !kOwnLaunch<QT, D>)) return rc;
  if constexpr (kOwnLaunch<QT, D>) {
    if (ta.splits == 1) {
      e = launch_pdl(kvq_prompt_exact_kernel<QT, D, BITS>, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, s, ta);
      if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
      return check_launch("kvq_attn");
    }
  }
  e = launch_pdl(kvq_prompt_join_kernel<QT, D, BITS>, dim3(static_cast<unsigned>(ta.items / ta.splits * (TQ / 16))), dim3(256), 0, s, ta);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "kvq_attn: %s", cudaGetErrorString(e));
  return check_launch("kvq_attn");
}

// Ranges of an item's tiles: as many as fill the SMs, where there are fewer items; a range has four tiles at least.
int splits_of(int64_t items, int64_t tiles) {
  const int64_t want = sm_count() / items, most = tiles / 4;
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : static_cast<int>(n);
}
int64_t wide_ints(int64_t items) { return (items + 3) / 4 * 4; }
int64_t row_items(int64_t B, int Hk, int64_t rows) { return B * Hk * ((rows + TQ - 1) / TQ); }

}  // namespace

int64_t attn_tc_bytes(int64_t B, int Hk, int D, int64_t rows) {
  const int64_t items = row_items(B, Hk, rows), splits = splits_of(items, INT32_MAX);
  return static_cast<int64_t>(sm_count()) * TQ * D * 4 + wide_ints(items * splits) * 4 + (splits > 1 ? items * splits * TQ * (D + 2) * 4 : 0);
}

int attn_tc(const AttnArgs& a, int dtype, int bits, int D, cudaStream_t s) {
  TcArgs ta;
  ta.a = a;
  const int64_t rows = static_cast<int64_t>(a.T) * a.group, items = row_items(a.c.B, a.c.Hk, rows);
  int64_t tiles = (a.c.capacity + KT - 1) / KT;        // the most that an item can have
  if (a.pos == nullptr) tiles = (a.pos_all + a.T + KT - 1) / KT;
  if (a.window > 0) tiles = min(tiles, (static_cast<int64_t>(a.window) + a.T + a.sinks) / KT + 3);
  ta.rows = static_cast<int>(rows);
  ta.row_tiles = static_cast<int>((rows + TQ - 1) / TQ);
  ta.splits = splits_of(items, tiles);
  CTDK_REQUIRE(rows <= INT32_MAX / 2 && items * ta.splits <= INT32_MAX / 16, "kvq_attn: too many rows");
  ta.items = static_cast<int>(items * ta.splits);
  ta.x64 = 0x64006400u;
  ta.total = a.part;                                   // (used by fp32 calls)
  ta.wide = reinterpret_cast<int*>(a.part + static_cast<int64_t>(sm_count()) * TQ * D);
  ta.a.part = reinterpret_cast<float*>(ta.wide + wide_ints(ta.items));
  const bool f32 = dtype == CTDK_DTYPE_F32;
  if (bits == 4) {
    if (D == 64) return f32 ? launch<float, 64, 4>(ta, s) : launch<__nv_bfloat16, 64, 4>(ta, s);
    return f32 ? launch<float, 128, 4>(ta, s) : launch<__nv_bfloat16, 128, 4>(ta, s);
  }
  if (D == 64) return f32 ? launch<float, 64, 8>(ta, s) : launch<__nv_bfloat16, 64, 8>(ta, s);
  return f32 ? launch<float, 128, 8>(ta, s) : launch<__nv_bfloat16, 128, 8>(ta, s);
}

}  // namespace kvq
}  // namespace ctdk
