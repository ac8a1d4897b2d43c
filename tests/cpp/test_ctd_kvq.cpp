// The quantised KV cache of the C++ surface (ops::QuantizedKV, nn::KVCache::allocate_quantized): attention over it against the
// attention written out on the host in 64 bits over the values that the cache gives back, and its refusals. With the
// argument "host" only the refusals that need no GPU run. Prints one "[ OK ]"/"[FAIL]" line per case and exits
// non-zero when any case failed.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "ctd/nn/attention.h"
#include "ctd/nn/kv_cache.h"
#include "ctd/ops/kv_cache.h"
#include "ctd/tensor.h"

using namespace ctd;

namespace {

int g_fail = 0, g_cases = 0, g_bad = 0;
#define CHECK(COND)                                                            \
  do {                                                                         \
    if (!(COND)) {                                                             \
      std::printf("    %s:%d: CHECK(%s) failed\n", __FILE__, __LINE__, #COND); \
      ++g_fail;                                                                \
    }                                                                          \
  } while (0)
#define CHECK_THROWS(EXPR)                                                 \
  do {                                                                     \
    bool threw_ = false;                                                   \
    try {                                                                  \
      (void)(EXPR);                                                        \
    } catch (const std::runtime_error&) {                                  \
      threw_ = true;                                                       \
    }                                                                      \
    if (!threw_) {                                                         \
      std::printf("    %s:%d: no throw: %s\n", __FILE__, __LINE__, #EXPR); \
      ++g_fail;                                                            \
    }                                                                      \
  } while (0)

template <typename F>
void run(const std::string& name, F fn) {
  const int before = g_fail;
  ++g_cases;
  try {
    fn();
  } catch (const std::exception& e) {
    std::printf("    exception: %s\n", e.what());
    ++g_fail;
  }
  std::printf("%s %s\n", g_fail == before ? "[ OK ]" : "[FAIL]", name.c_str());
  g_bad += g_fail != before;
}

std::vector<float> noise(size_t n, unsigned seed, float scale = 1.0f) {
  std::mt19937 g(seed);
  std::normal_distribution<float> d(0.0f, scale);
  std::vector<float> x(n);
  for (float& v : x) v = d(g);
  return x;
}
Tensor dev(const std::vector<float>& x, std::vector<int64_t> shape) { return Tensor::from_host(x.data(), std::move(shape), DType::kFloat32, kCUDA0); }
std::vector<float> host(const Tensor& t) {
  std::vector<float> x(static_cast<size_t>(t.numel()));
  t.copy_to_host(x.data());
  return x;
}

struct Sizes {
  int64_t B, T, H, Hk, D, pos, window, sinks;
  int bits;
};

nn::Attention layer(const Sizes& z, int64_t hid) {
  nn::Attention a;
  const float s = 1.0f / std::sqrt(static_cast<float>(hid));
  a.q_proj = nn::Linear{dev(noise(z.H * z.D * hid, 1, s), {z.H * z.D, hid})};
  a.k_proj = nn::Linear{dev(noise(z.Hk * z.D * hid, 2, s), {z.Hk * z.D, hid})};
  a.v_proj = nn::Linear{dev(noise(z.Hk * z.D * hid, 3, s), {z.Hk * z.D, hid})};
  a.o_proj = nn::Linear{dev(noise(hid * z.H * z.D, 4, s), {hid, z.H * z.D})};
  a.num_heads = static_cast<int>(z.H);
  a.num_kv_heads = static_cast<int>(z.Hk);
  a.head_dim = static_cast<int>(z.D);
  return a;
}

// What attention over keys and values k, v [B, Hk, L, D] gives the queries [B, T, H, D] at pos .. pos + T - 1, in 64 bits.
std::vector<double> plain(const std::vector<float>& q, const std::vector<float>& k, const std::vector<float>& v, const Sizes& z) {
  const int64_t L = z.pos + z.T;
  std::vector<double> out(q.size(), 0.0), p(L);
  for (int64_t b = 0; b < z.B; ++b)
    for (int64_t t = 0; t < z.T; ++t)
      for (int64_t h = 0; h < z.H; ++h) {
        const float* qr = &q[((b * z.T + t) * z.H + h) * z.D];
        const int64_t head = (b * z.Hk + h / (z.H / z.Hk)) * L, i = z.pos + t;
        double top = -INFINITY, sum = 0.0;
        for (int64_t j = 0; j < L; ++j) {
          const bool seen = j <= i && (z.window == 0 || i - j < z.window || j < z.sinks);
          double s = 0.0;
          for (int64_t d = 0; d < z.D; ++d) s += static_cast<double>(qr[d]) * k[(head + j) * z.D + d];
          p[j] = seen ? s / std::sqrt(static_cast<double>(z.D)) : -INFINITY;
          top = std::max(top, p[j]);
        }
        for (int64_t j = 0; j < L; ++j) sum += p[j] = std::exp(p[j] - top);
        for (int64_t j = 0; j < L; ++j)
          for (int64_t d = 0; d < z.D; ++d) out[((b * z.T + t) * z.H + h) * z.D + d] += p[j] / sum * v[(head + j) * z.D + d];
      }
  return out;
}

// nn::Attention over a quantised cache, a prompt and then single tokens: its context is what the layer's own queries give, in 64
// bits, over the values read back; the projections around it are the layer's own.
void attends(const Sizes& z) {
  const int64_t hid = 96;
  const nn::Attention a = layer(z, hid);
  nn::KVCache cache = nn::KVCache::allocate_quantized(1, a.num_kv_heads, a.head_dim, z.B, z.pos + z.T + 3, z.bits, kCUDA0, z.window, z.sinks);
  CHECK(cache.layers[0].quantized.capacity() % 64 == 0 && cache.layers[0].quantized.capacity() >= z.pos + z.T + 3);
  // what came before
  if (z.pos > 0) a.forward(dev(noise(z.B * z.pos * hid, 5), {z.B, z.pos, hid}), &cache.layers[0], 0);
  Sizes now = z;
  for (int step = 0; step < 3; ++step) {
    const Tensor x = dev(noise(z.B * now.T * hid, 6 + step), {z.B, now.T, hid});
    const Tensor got = a.forward(x, &cache.layers[0], static_cast<int>(now.pos));
    Tensor q = a.q_proj.forward(x).reshape({z.B, now.T, z.H, z.D});
    ops::apply_rope_inplace(q, static_cast<int>(now.pos), a.rope_theta, a.rope_scaling);
    const auto kv = ops::read_kv_quantized(cache.layers[0].quantized, now.pos + now.T, 1);
    const std::vector<double> want = plain(host(q), host(kv.first), host(kv.second), now);
    const std::vector<float> ctx = host(ops::attention_quantized(q, cache.layers[0].quantized, now.pos));
    double worst = 0.0, most = 0.0;
    for (size_t i = 0; i < want.size(); ++i) {
      worst = std::max(worst, std::fabs(ctx[i] - want[i]));
      most = std::max(most, std::fabs(want[i]));
    }
    // scores of a few units, held with 22 bits, err by some 2^-20, and the sums of the products round a few hundred times
    // at 2^-24: 1e-5 of the largest value is ten times that
    CHECK(worst <= 1e-5 * most);
    // the layer ends with its own projection of that context
    const std::vector<float> projected = host(a.o_proj.forward(dev(ctx, {z.B, now.T, z.H * z.D}))), y = host(got);
    CHECK(projected == y);
    now.pos += now.T;
    now.T = 1;
  }
}

// The values come back within half a step of the format, from fp32 and expanded over the group.
void reads_back(int bits) {
  const int64_t B = 2, T = 5, Hk = 2, D = 64, pos = 61;
  ops::QuantizedKV c = ops::QuantizedKV::allocate(Hk, D, B, 66, bits, kCUDA0);
  const std::vector<float> k = noise(B * T * Hk * D, 20), v = noise(B * T * Hk * D, 21);
  ops::write_kv_quantized(c, dev(k, {B, T, Hk, D}), dev(v, {B, T, Hk, D}), pos);
  const auto kv = ops::read_kv_quantized(c, pos + T, 3);
  const std::vector<float> gk = host(kv.first), gv = host(kv.second);
  for (int64_t b = 0; b < B; ++b)
    for (int64_t t = 0; t < T; ++t)
      for (int64_t h = 0; h < Hk * 3; ++h)
        for (int64_t d = 0; d < D; ++d) {
          const int64_t from = ((b * T + t) * Hk + h / 3) * D, to = ((b * Hk * 3 + h) * (pos + T) + pos + t) * D + d;
          float ak = 0.0f, av = 0.0f;
          for (int64_t e = d / 32 * 32; e < d / 32 * 32 + 32; ++e) {
            ak = std::max(ak, std::fabs(k[from + e]));
            av = std::max(av, std::fabs(v[from + e]));
          }
          // half a step; a step is 1/7 (1/127) of the largest magnitude, rounded up by at most 1/8 (by less than twice)
          const float half = bits == 4 ? 0.5f / 7.0f * 1.126f : 0.5f / 127.0f * 2.001f;
          CHECK(std::fabs(gk[to] - k[from + d]) <= half * ak);
          CHECK(std::fabs(gv[to] - v[from + d]) <= half * av);
        }
}

void refusals_without_gpu() {
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, 1, 64, 5, kCUDA0));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 48, 1, 64, 4, kCUDA0));
  CHECK_THROWS(ops::QuantizedKV::allocate(0, 64, 1, 64, 4, kCUDA0));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, 1, 0, 4, kCUDA0));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, -1, 64, 4, kCUDA0));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, 1, 64, 4, kCUDA0, -1));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, 1, 64, 4, kCUDA0, 8, -1));
  CHECK_THROWS(ops::QuantizedKV::allocate(2, 64, 1, 64, 4, kCPU));
  CHECK_THROWS(nn::KVCache::allocate_quantized(3, 2, 64, 1, 64, 3, kCUDA0));
  ops::QuantizedKV none;
  const Tensor x = Tensor::zeros({1, 1, 2, 64}, DType::kFloat32, kCPU);
  CHECK_THROWS(ops::write_kv_quantized(none, x, x, 0));
  CHECK_THROWS(ops::read_kv_quantized(none, 0, 1));
  CHECK_THROWS(ops::attention_quantized(x, none, 0));
}

void refusals() {
  ops::QuantizedKV c = ops::QuantizedKV::allocate(2, 64, 1, 60, 8, kCUDA0);
  auto t = [](std::vector<int64_t> shape, DType d = DType::kFloat32) { return Tensor::zeros(std::move(shape), d, kCUDA0); };
  const Tensor ok = t({1, 2, 2, 64});
  ops::write_kv_quantized(c, ok, ok, 62);
  CHECK_THROWS(ops::write_kv_quantized(c, ok, ok, 63));
  CHECK_THROWS(ops::write_kv_quantized(c, ok, ok, -1));
  CHECK_THROWS(ops::write_kv_quantized(c, ok, t({1, 1, 2, 64}), 0));
  CHECK_THROWS(ops::write_kv_quantized(c, ok, t({1, 2, 2, 64}, DType::kBFloat16), 0));
  CHECK_THROWS(ops::write_kv_quantized(c, t({1, 2, 3, 64}), t({1, 2, 3, 64}), 0));
  CHECK_THROWS(ops::write_kv_quantized(c, t({2, 2, 2, 64}), t({2, 2, 2, 64}), 0));
  CHECK_THROWS(ops::write_kv_quantized(c, t({1, 2, 2, 128}), t({1, 2, 2, 128}), 0));
  CHECK_THROWS(ops::write_kv_quantized(c, t({2, 2, 64}), t({2, 2, 64}), 0));
  CHECK_THROWS(ops::read_kv_quantized(c, 65, 1));
  CHECK_THROWS(ops::read_kv_quantized(c, 1, 0));
  CHECK_THROWS(ops::read_kv_quantized(c, 1, 1, DType::kFloat16));
  CHECK_THROWS(ops::attention_quantized(t({1, 1, 3, 64}), c, 0));
  CHECK_THROWS(ops::attention_quantized(t({1, 1, 2, 64}), c, 64));
  CHECK_THROWS(ops::attention_quantized(t({1, 1, 2, 64}, DType::kFloat16), c, 0));
  CHECK(ops::read_kv_quantized(c, 0, 1).first.numel() == 0);
}

}  // namespace

int main(int argc, char** argv) {
  run("refusals_without_gpu", refusals_without_gpu);
  if (argc < 2 || std::strcmp(argv[1], "host") != 0) {
    run("refusals", refusals);
    for (int bits : {4, 8}) {
      run("reads_back_" + std::to_string(bits), [&] { reads_back(bits); });
      run("tokens_after_a_prompt_" + std::to_string(bits), [&] { attends({2, 70, 4, 2, 64, 0, 0, 0, bits}); });
      run("window_and_sinks_" + std::to_string(bits), [&] { attends({1, 40, 6, 2, 128, 130, 50, 3, bits}); });
    }
  }
  std::printf("%d cases, %d failed\n", g_cases, g_bad);
  return g_bad ? 1 : 0;
}
