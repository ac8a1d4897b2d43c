// What the two attention kernels over the quantised cache share (kv_quant_attn.cu: few query rows a key/value head;
// kv_quant_attn_tc.cu: prompts): their arguments, and which tiles of positions a block of query rows has to visit.
#pragma once

#include "kv_quant.cuh"

namespace ctdk {
namespace kvq {

struct AttnArgs {
  Cache c;
  const void* q;                         // row t of sequence b at b * batch_stride + t * row_stride, heads side by side
  void* out;                             // [B, T, H, D]
  int64_t row_stride, batch_stride;
  const int32_t *pos, *count;
  int64_t pos_all;
  int window, sinks;                     // 0: no window
  int T, H, group;                       // group: query heads of a key/value head
  float scale_log2;                      // scale * log2(e)
  float* part;                           // partial results (kv_quant_attn.cu)
  int* status;
};

// The positions that a block of query rows visits, as tiles of `tile` positions: first the ones that hold sinks, then the
// ones from the first row's window up to the last row.
struct Visit {
  int lo_row, hi_row;                    // positions of its first and behind its last valid row; none: 0, 0
  int sink_tiles, win_tile, tiles;
  __host__ __device__ __forceinline__ int tile_at(int k) const { return k < sink_tiles ? k : win_tile + (k - sink_tiles); }
};

// pos, count: of the sequence; the block has its rows t0 .. t0 + rows - 1. A row is valid if it is one of the sequence's new rows
// and its position is one of the cache's.
__host__ __device__ __forceinline__ Visit visit_of(int64_t pos, int64_t count, int64_t t0, int64_t rows, int64_t capacity, int64_t window,
                                                   int64_t sinks, int tile) {
  const int64_t n = count - t0 < rows ? count - t0 : rows, first = pos + t0;
  const int64_t a = first > 0 ? first : 0, e = first + n < capacity ? first + n : capacity;
  Visit v = {0, 0, 0, 0, 0};
  if (n <= 0 || e <= a) return v;
  v.lo_row = static_cast<int>(a);
  v.hi_row = static_cast<int>(e);
  const int64_t lo = window > 0 && a >= window ? a - window + 1 : 0;
  v.win_tile = static_cast<int>(lo / tile);
  const int st = static_cast<int>(((sinks < e ? sinks : e) + tile - 1) / tile);
  v.sink_tiles = window <= 0 ? 0 : (st < v.win_tile ? st : v.win_tile);
  v.tiles = v.sink_tiles + static_cast<int>((e + tile - 1) / tile) - v.win_tile;
  return v;
}

#ifdef __CUDACC__
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// As mbar_wait_bounded_w of common.cuh, with a time for which the hardware may put the warp to sleep, and with what follows a first
// try that fails off the common path: the kernels' roles together are larger than an instruction cache, and most waits are over at once.
__device__ __forceinline__ uint32_t try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.b32 %0, 1, 0, p;\n}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
               : "memory");
  return ok;
}
__device__ __forceinline__ bool wait_longer(uint64_t* bar, uint32_t parity, int* status, int where) {
  const uint64_t since = globaltimer_ns();
  uint32_t ok;
  for (int tries = 0; (ok = try_wait(bar, parity)) == 0; ++tries)
    if ((tries & 15) == 15 && globaltimer_ns() - since > kWaitBudgetNs) {
      if (status != nullptr && atomicCAS(status, 0, CTDK_ETIMEOUT) == 0) {
        status[1] = where;
        status[2] = static_cast<int>(blockIdx.x);
        status[3] = static_cast<int>(parity);
      }
      break;
    }
  return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ bool wait_w(uint64_t* bar, uint32_t parity, int* status, int where) {
  bool ok = __all_sync(0xffffffffu, try_wait(bar, parity) != 0);
  if (__builtin_expect(!ok, 0)) ok = wait_longer(bar, parity, status, where);
  return ok;
}
// As bulk_load of common.cuh, without a cache hint.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
// Position of row t of a sequence, or -1 if it is not valid.
__device__ __forceinline__ int row_position(int64_t pos, int64_t count, int64_t t, int64_t capacity) {
  const int64_t i = pos + t;
  return t < count && i >= 0 && i < capacity ? static_cast<int>(i) : -1;
}
// Whether the query at position i (-1: none) sees position j; w, s: window (0: none) and sinks.
__device__ __forceinline__ bool sees(int i, int j, int w, int s) { return j <= i && (w == 0 || i - j < w || j < s); }
#endif

int check_cache(const ctdk_kvq_cache* c, const char* what);   // kv_quant.cu
// kv_quant_attn_tc.cu: prompts, in a workspace (a.part) of attn_tc_bytes for rows = T * group.
int64_t attn_tc_bytes(int64_t B, int Hk, int D, int64_t rows);
int attn_tc(const AttnArgs& a, int dtype, int bits, int D, cudaStream_t s);

}  // namespace kvq
}  // namespace ctdk
