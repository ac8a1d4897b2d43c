// Writing rows into a key/value cache of 4 or 8 bits, and reading them back (layout: kv_quant.cuh). Beside the
// fp32 cache's ctdk_kv_write / ctdk_kv_read_expanded (emberlm src/ops/kv_cache.cu:14-109).
//
// A thread takes sixteen neighbouring values, two threads a group; a row's threads are neighbours and consecutive rows
// are consecutive positions of one head, so that the cache side is contiguous and the other side comes in whole head
// rows of 128 to 512 bytes. (With eight values a thread the index arithmetic, not memory, was the limit.)
// Measured (B200, copy bandwidth 6.45 TB/s): 4 x 4096 rows of 8 x 128, keys and values, one call after the other over more data than
// L2 holds, us and TB/s:
//             fp32, 4 bits   bfloat16, 4 bits   fp32, 8 bits   bfloat16, 8 bits
//   write     33.0  4.6      30.7  2.8          28.2  6.0      22.7  4.5
//   read      32.6  4.7      21.6  4.0          33.4  5.1      20.6  5.0
// Writing 4 bits spends its time on the exact rounding (a quotient with its remainder a value, from bfloat16 rows too, which would need
// less); the others run at 62 to 93 % of the copy bandwidth.
#include "kv_quant.cuh"

namespace ctdk {
namespace kvq {
namespace {

constexpr int kThreads = 256;

struct RowArgs {
  const void* src[2];
  int64_t row_stride, batch_stride;      // elements between tokens, between sequences
  uint8_t* codes[2];
  __nv_bfloat16* scales[2];
  const int32_t *pos, *count;            // per sequence, or null
  int64_t pos_all, capacity;
  int64_t rows;                          // B * Hk * T
  int T, Hk;
};

// Eight 4-bit codes for the scale s, each value to the nearest whole number of steps, half to even, decided exactly, packed as they
// are stored. The quotient is corrected once by its remainder (exact: both terms are whole multiples of the smaller one's last place
// and their difference is short), which makes it exact wherever it is a half, a common case of bfloat16 values; adding 1.5 * 2^23
// (+ 8: the low bits are the code) rounds it. What is left are fp32 values so close to a half that the quotient rounds to it: they end
// up further than half a step away, and 64 bits decide, where a quotient of 24 bits by 4 cannot be mistaken for a half.
// (Conversions to integers run at a sixteenth of the rate.)
__device__ __forceinline__ uint32_t nearest8(const float (&x)[8], float s, float inv) {   // inv: 1 / s, rounded
  const float magic = 12582912.0f + 8.0f;
  uint32_t w = 0;
  float far = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float q0 = __fmul_rn(x[k], inv), q = __fmaf_rn(__fmaf_rn(-q0, s, x[k]), inv, q0);
    const float y = __fadd_rn(q, magic), n = __fadd_rn(y, -magic);
    far = fmaxf(far, fabsf(__fmaf_rn(-n, s, x[k])));
    w |= (__float_as_uint(y) & 0xfu) << (4 * k);
  }
  if (far <= 0.5f * s) return w;
  w = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) w |= static_cast<uint32_t>(static_cast<int>(rint(static_cast<double>(x[k]) / s)) + 8) << (4 * k);
  return w;
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kThreads) kvq_write_kernel(const RowArgs a) {
  constexpr int kPerRow = D / 16, kRowBytes = D * BITS / 8;
  constexpr float kPart = 1.0f / (BITS == 4 ? 7.0f : 127.0f);
  constexpr int kCut = BITS == 4 ? 20 : 23;   // low bits of the fp32 scale that rounding up clears
  pdl_launch();
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, r = i / kPerRow;
  const int lane16 = static_cast<int>(i % kPerRow), which = blockIdx.y;
  bool live = r < a.rows;
  float x[2][8] = {};
  int64_t at = 0;
  if (live) {
    const int64_t bh = quotient(r, a.T);
    const int t = static_cast<int>(r - bh * a.T);
    const int64_t b = quotient(bh, a.Hk);
    const int h = static_cast<int>(bh - b * a.Hk);
    const int64_t p = (a.pos != nullptr ? static_cast<int64_t>(a.pos[b]) : a.pos_all) + t;
    live = p >= 0 && p < a.capacity && (a.count == nullptr || t < a.count[b]);
    at = bh * a.capacity + p;
    if (live) {
      const T* src = static_cast<const T*>(which ? a.src[1] : a.src[0]) + b * a.batch_stride + t * a.row_stride + h * D + lane16 * 16;
      load8(src, x[0]);
      load8(src + 8, x[1]);
    }
  }
  float most = 0.0f;
  bool nan = false;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    most = fmaxf(most, fabsf(x[k / 8][k % 8]));
    nan |= isnan(x[k / 8][k % 8]);
  }
  if (nan) most = __int_as_float(0x7f800000);
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
  if (!live) return;
  const bool fine = most < kMost;
  float s = __uint_as_float(((__float_as_uint(__fmul_rn(most, kPart)) + ((1u << kCut) - 1u)) >> kCut) << kCut);
  uint8_t* dst = (which ? a.codes[1] : a.codes[0]) + at * kRowBytes + lane16 * 2 * BITS;
  if (!fine) s = __int_as_float(0x7fc00000);
  const bool none = !fine || s == 0.0f;                // every code 0
  if constexpr (BITS == 8) {
    const float inv = none ? 0.0f : __fdiv_rn(1.0f, s);   // a power of two from 2^-126 on: exact, and so is the product
    uint32_t u[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) u[k] = none ? 128u : __float_as_uint(__fmaf_rn(x[k / 8][k % 8], inv, 12582912.0f + 128.0f));
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = prmt(prmt(u[4 * k], u[4 * k + 1], 0x40), prmt(u[4 * k + 2], u[4 * k + 3], 0x40), 0x5410);
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[2] = {0x88888888u, 0x88888888u};
    if (!none && s >= 0x1p-100f) {
      const float inv = __fdiv_rn(1.0f, s);
      w[0] = nearest8(x[0], s, inv);
      w[1] = nearest8(x[1], s, inv);
    } else if (!none) {                                // a reciprocal could overflow
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        w[v] = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[v] |= static_cast<uint32_t>(static_cast<int>(fmin(fmax(rint(static_cast<double>(x[v][k]) / s), -7.0), 7.0)) + 8) << (4 * k);
      }
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
  if ((lane16 & 1) == 0)
    (which ? a.scales[1] : a.scales[0])[at * (D / kGroup) + lane16 / 2] = __ushort_as_bfloat16(static_cast<unsigned short>(__float_as_uint(s) >> 16));
}

struct ReadArgs {
  Cache c;
  void* out[2];                          // [B, Hk * group, length, D]
  int64_t start, length, rows;           // rows = B * Hk * length
  int group;
};

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {   // exact
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// Values of a thread that reads: 32 bytes of output (with 64 its stores, whole sectors apart, measured a fifth slower).
template <typename T>
constexpr int kReadBy = sizeof(T) == 4 ? 8 : 16;

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kThreads) kvq_read_kernel(const ReadArgs a) {
  constexpr int kBy = kReadBy<T>, kPerRow = D / kBy, kRowBytes = D * BITS / 8, kWords = kBy * BITS / 32;
  pdl_launch();
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, r = i / kPerRow;
  const int place = static_cast<int>(i % kPerRow), which = blockIdx.y;
  if (r >= a.rows) return;
  const int64_t bh = quotient(r, a.length), t = r - bh * a.length, at = bh * a.c.capacity + a.start + t;
  const float s = __bfloat162float((which ? a.c.scales[1] : a.c.scales[0])[at * (D / kGroup) + place * kBy / kGroup]);
  const uint8_t* src = (which ? a.c.codes[1] : a.c.codes[0]) + at * kRowBytes + place * kBy * BITS / 8;
  uint32_t w[kWords];
  if constexpr (kWords == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(src));
  }
  // The code's bits under the exponent of a power of two, whose multiple of the scale the same operation takes off: exact.
  const float b = s * (BITS == 8 ? -32896.0f : -136.0f);   // (2^15 + 128) s, (2^7 + 8) s
  float x[kBy / 8][8];
#pragma unroll
  for (int k = 0; k < kBy; ++k) {
    uint32_t u;
    if constexpr (BITS == 8) {
      u = prmt(w[k / 4], 0x47000000u, 0x7604u | (k % 4) << 4);
    } else {
      const int n = k % 8;
      u = ((n < 4 ? w[k / 8] << (16 - 4 * n) : w[k / 8] >> (4 * n - 16)) & 0x000f0000u) | 0x43000000u;
    }
    x[k / 8][k % 8] = fmaf(__uint_as_float(u), s, b);
  }
  T* dst = static_cast<T*>(which ? a.out[1] : a.out[0]) + (bh * a.group * a.length + t) * D + place * kBy;
  for (int g = 0; g < a.group; ++g)
#pragma unroll
    for (int v = 0; v < kBy / 8; ++v) store8(dst + g * a.length * D + 8 * v, x[v]);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename K, typename A>
int launch_rows(K kernel, const A& a, int64_t rows, int per_row, cudaStream_t s, const char* what) {   // threads of a row
  const int64_t blocks = (rows * per_row + kThreads - 1) / kThreads;
  CTDK_REQUIRE(blocks <= INT32_MAX, "%s: too many rows", what);
  const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(blocks), 2), dim3(kThreads), 0, s, a);
  if (e != cudaSuccess) return fail(CTDK_ELAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace

int check_cache(const ctdk_kvq_cache* c, const char* what) {
  CTDK_REQUIRE(c != nullptr, "%s: no cache", what);
  CTDK_REQUIRE(c->bits == 4 || c->bits == 8, "%s: bits must be 4 or 8", what);
  CTDK_REQUIRE(c->D == 64 || c->D == 128, "%s: D must be 64 or 128", what);
  CTDK_REQUIRE(c->B >= 0 && c->B <= INT32_MAX && c->Hk > 0, "%s: bad batch or head count", what);
  CTDK_REQUIRE(c->capacity > 0 && c->capacity % kCapacityStep == 0 && c->capacity <= INT32_MAX - 2 * kCapacityStep,
               "%s: capacity must be a multiple of %d below 2^31", what, kCapacityStep);
  if (c->B == 0) return CTDK_OK;
  CTDK_REQUIRE(c->k_codes != nullptr && c->k_scales != nullptr && c->v_codes != nullptr && c->v_scales != nullptr, "%s: null cache pointer", what);
  CTDK_REQUIRE(aligned(c->k_codes, 16) && aligned(c->k_scales, 16) && aligned(c->v_codes, 16) && aligned(c->v_scales, 16),
               "%s: the cache's pointers must be 16-byte aligned", what);
  return CTDK_OK;
}

}  // namespace kvq
}  // namespace ctdk

using namespace ctdk;

extern "C" {

int ctdk_kvq_write(const ctdk_kvq_cache* cache, const void* k, const void* v, int dtype, int64_t row_stride, int64_t batch_stride, int64_t T,
                   const int32_t* pos, int64_t pos_all, const int32_t* count, void* stream) {
  if (const int rc = kvq::check_cache(cache, "kvq_write"); rc != CTDK_OK) return rc;
  CTDK_REQUIRE(dtype == CTDK_DTYPE_F32 || dtype == CTDK_DTYPE_BF16, "kvq_write: dtype must be CTDK_DTYPE_F32 or CTDK_DTYPE_BF16");
  CTDK_REQUIRE(T >= 0 && T <= INT32_MAX, "kvq_write: bad T");
  CTDK_REQUIRE(pos != nullptr || (pos_all >= 0 && pos_all <= cache->capacity - T), "kvq_write: %lld positions from %lld on exceed the capacity %lld",
               static_cast<long long>(T), static_cast<long long>(pos_all), static_cast<long long>(cache->capacity));
  if (T == 0 || cache->B == 0) return CTDK_OK;
  const int64_t unit = dtype == CTDK_DTYPE_F32 ? 4 : 8;   // elements in 16 bytes
  CTDK_REQUIRE(k != nullptr && v != nullptr && kvq::aligned(k, 16) && kvq::aligned(v, 16), "kvq_write: k and v must be 16-byte aligned");
  CTDK_REQUIRE(row_stride % unit == 0 && batch_stride % unit == 0 && row_stride >= 0 && batch_stride >= 0,
               "kvq_write: strides must be multiples of 16 bytes");
  kvq::RowArgs a;
  a.src[0] = k;
  a.src[1] = v;
  a.row_stride = row_stride;
  a.batch_stride = batch_stride;
  a.codes[0] = static_cast<uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<uint8_t*>(cache->v_codes);
  a.scales[0] = static_cast<__nv_bfloat16*>(cache->k_scales);
  a.scales[1] = static_cast<__nv_bfloat16*>(cache->v_scales);
  a.pos = pos;
  a.count = count;
  a.pos_all = pos_all;
  a.capacity = cache->capacity;
  a.rows = cache->B * cache->Hk * T;
  a.T = static_cast<int>(T);
  a.Hk = cache->Hk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32 = dtype == CTDK_DTYPE_F32;
  auto go = [&](auto* kernel) { return kvq::launch_rows(kernel, a, a.rows, cache->D / 16, s, "kvq_write"); };
  if (cache->bits == 4) {
    if (cache->D == 64) return f32 ? go(kvq::kvq_write_kernel<float, 4, 64>) : go(kvq::kvq_write_kernel<__nv_bfloat16, 4, 64>);
    return f32 ? go(kvq::kvq_write_kernel<float, 4, 128>) : go(kvq::kvq_write_kernel<__nv_bfloat16, 4, 128>);
  }
  if (cache->D == 64) return f32 ? go(kvq::kvq_write_kernel<float, 8, 64>) : go(kvq::kvq_write_kernel<__nv_bfloat16, 8, 64>);
  return f32 ? go(kvq::kvq_write_kernel<float, 8, 128>) : go(kvq::kvq_write_kernel<__nv_bfloat16, 8, 128>);
}

int ctdk_kvq_read(const ctdk_kvq_cache* cache, int64_t start, int64_t length, int group, int dtype, void* k_out, void* v_out, void* stream) {
  if (const int rc = kvq::check_cache(cache, "kvq_read"); rc != CTDK_OK) return rc;
  CTDK_REQUIRE(dtype == CTDK_DTYPE_F32 || dtype == CTDK_DTYPE_BF16, "kvq_read: dtype must be CTDK_DTYPE_F32 or CTDK_DTYPE_BF16");
  CTDK_REQUIRE(start >= 0 && length >= 0 && start <= cache->capacity - length, "kvq_read: positions out of range");
  CTDK_REQUIRE(group > 0, "kvq_read: group must be > 0");
  if (length == 0 || cache->B == 0) return CTDK_OK;
  CTDK_REQUIRE(k_out != nullptr && v_out != nullptr && kvq::aligned(k_out, 16) && kvq::aligned(v_out, 16),
               "kvq_read: outputs must be 16-byte aligned");
  kvq::ReadArgs a;
  a.c = kvq::Cache{{static_cast<const uint8_t*>(cache->k_codes), static_cast<const uint8_t*>(cache->v_codes)},
                   {static_cast<const __nv_bfloat16*>(cache->k_scales), static_cast<const __nv_bfloat16*>(cache->v_scales)},
                   cache->capacity, static_cast<int>(cache->B), cache->Hk};
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.start = start;
  a.length = length;
  a.rows = cache->B * cache->Hk * length;
  a.group = group;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32 = dtype == CTDK_DTYPE_F32;
  auto go = [&](auto* kernel) { return kvq::launch_rows(kernel, a, a.rows, cache->D / (f32 ? kvq::kReadBy<float> : kvq::kReadBy<__nv_bfloat16>), s, "kvq_read"); };
  if (cache->bits == 4) {
    if (cache->D == 64) return f32 ? go(kvq::kvq_read_kernel<float, 4, 64>) : go(kvq::kvq_read_kernel<__nv_bfloat16, 4, 64>);
    return f32 ? go(kvq::kvq_read_kernel<float, 4, 128>) : go(kvq::kvq_read_kernel<__nv_bfloat16, 4, 128>);
  }
  if (cache->D == 64) return f32 ? go(kvq::kvq_read_kernel<float, 8, 64>) : go(kvq::kvq_read_kernel<__nv_bfloat16, 8, 64>);
  return f32 ? go(kvq::kvq_read_kernel<float, 8, 128>) : go(kvq::kvq_read_kernel<__nv_bfloat16, 8, 128>);
}

}  // extern "C"
