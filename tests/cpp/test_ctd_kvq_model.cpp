// nn::Model over a quantised KV cache (nn::KVCache::allocate_quantized): Model::forward gives what its own layers give one after the
// other over a second cache, for a prompt, a longer piece and single tokens, and leaves the same bytes in the cache; and empty calls.
// Prints one "[ OK ]"/"[FAIL]" line per case and exits non-zero when any case failed.
#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "ctd/nn/kv_cache.h"
#include "ctd/nn/model.h"
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

nn::LlamaConfig config(int head_dim, bool qk_norm) {
  nn::LlamaConfig c{};
  c.vocab_size = 320;
  c.hidden_size = 128;
  c.intermediate_size = 256;
  c.num_hidden_layers = 3;
  c.num_attention_heads = 4;
  c.num_key_value_heads = 2;
  c.head_dim = head_dim;
  c.max_position_embeddings = 512;
  c.rms_norm_eps = 1e-5f;
  c.rope_theta = 10000.0f;
  c.tie_word_embeddings = true;
  c.qk_norm = qk_norm;
  return c;
}

nn::Model model(const nn::LlamaConfig& c, unsigned seed) {
  std::mt19937 rng(seed);
  TensorDict w;
  auto put = [&](const std::string& name, std::vector<int64_t> shape, float mean, float spread) {
    std::normal_distribution<float> nd(mean, spread);
    size_t n = 1;
    for (int64_t d : shape) n *= static_cast<size_t>(d);
    std::vector<float> h(n);
    for (float& v : h) v = nd(rng);
    w[name] = Tensor::from_host(h.data(), std::move(shape), DType::kFloat32, kCPU);
  };
  const int64_t hid = c.hidden_size, I = c.intermediate_size, D = c.head_dim, H = c.num_attention_heads, Hk = c.num_key_value_heads;
  put("model.embed_tokens.weight", {c.vocab_size, hid}, 0.0f, 0.5f);
  for (int l = 0; l < c.num_hidden_layers; ++l) {
    const std::string p = "model.layers." + std::to_string(l) + ".";
    put(p + "input_layernorm.weight", {hid}, 1.0f, 0.1f);
    put(p + "self_attn.q_proj.weight", {H * D, hid}, 0.0f, 0.1f);
    put(p + "self_attn.k_proj.weight", {Hk * D, hid}, 0.0f, 0.1f);
    put(p + "self_attn.v_proj.weight", {Hk * D, hid}, 0.0f, 0.1f);
    put(p + "self_attn.o_proj.weight", {hid, H * D}, 0.0f, 0.1f);
    if (c.qk_norm) {
      put(p + "self_attn.q_norm.weight", {D}, 1.0f, 0.1f);
      put(p + "self_attn.k_norm.weight", {D}, 1.0f, 0.1f);
    }
    put(p + "post_attention_layernorm.weight", {hid}, 1.0f, 0.1f);
    put(p + "mlp.gate_proj.weight", {I, hid}, 0.0f, 0.1f);
    put(p + "mlp.up_proj.weight", {I, hid}, 0.0f, 0.1f);
    put(p + "mlp.down_proj.weight", {hid, I}, 0.0f, 0.1f);
  }
  put("model.norm.weight", {hid}, 1.0f, 0.1f);
  return nn::build_model(w, c);
}

template <typename T = float>
std::vector<T> host(const Tensor& t) {
  std::vector<T> h(static_cast<size_t>(t.nbytes()) / sizeof(T));
  t.copy_to_host(h.data());
  return h;
}

void generates(int head_dim, bool qk_norm, int bits, int64_t window, int64_t sinks) {
  const nn::LlamaConfig c = config(head_dim, qk_norm);
  const nn::Model m = model(c, 7);
  const int64_t B = 2, steps[] = {70, 9, 1, 1, 1};
  int64_t total = 0;
  for (int64_t t : steps) total += t;
  auto allocate = [&] {
    return nn::KVCache::allocate_quantized(c.num_hidden_layers, c.num_key_value_heads, c.head_dim, B, total, bits, kCUDA0, window, sinks);
  };
  nn::KVCache cache = allocate(), mine = allocate();
  std::mt19937 rng(8);
  std::uniform_int_distribution<int> token(0, c.vocab_size - 1);
  int64_t pos = 0;
  for (int64_t T : steps) {
    std::vector<int64_t> ids(static_cast<size_t>(B * T));
    for (int64_t& v : ids) v = token(rng);
    const Tensor input = Tensor::from_host(ids.data(), {B, T}, DType::kInt64, kCUDA0);
    const Tensor logits = m.forward(input, &cache, static_cast<int>(pos));
    Tensor h = m.embed_tokens.forward(input);
    for (size_t i = 0; i < m.layers.size(); ++i) {
      const nn::TransformerBlock& b = m.layers[i];
      h = ops::add(h, b.self_attn.forward(b.input_layernorm.forward(h), &mine.layers[i], static_cast<int>(pos)));
      h = ops::add(h, b.mlp.forward(b.post_attention_layernorm.forward(h)));
    }
    const Tensor want = nn::Linear{m.embed_tokens.weight}.forward(m.norm.forward(h));
    pos += T;
    CHECK(logits.shape() == (std::vector<int64_t>{B, T, c.vocab_size}));
    CHECK(host(logits) == host(want));
    bool finite = true;
    for (float x : host(logits)) finite = finite && std::isfinite(x);
    CHECK(finite);
    CHECK(cache.current_len == pos);
  }
  for (size_t i = 0; i < m.layers.size(); ++i) {
    const ops::QuantizedKV &a = cache.layers[i].quantized, &b = mine.layers[i].quantized;
    CHECK(host<int32_t>(a.k_codes) == host<int32_t>(b.k_codes) && host<int32_t>(a.v_codes) == host<int32_t>(b.v_codes));
    CHECK(host<uint16_t>(a.k_scales) == host<uint16_t>(b.k_scales) && host<uint16_t>(a.v_scales) == host<uint16_t>(b.v_scales));
    // layers have caches of their own
    if (i > 0) CHECK(host<int32_t>(a.k_codes) != host<int32_t>(cache.layers[i - 1].quantized.k_codes));
  }
}

// One token, a short and a long piece: no sequences, or no rows.
void empty_calls() {
  for (int64_t T : {int64_t{1}, int64_t{16}, int64_t{40}}) {
    ops::QuantizedKV none = ops::QuantizedKV::allocate(2, 64, 0, 64, 4, kCUDA0);
    const Tensor x = Tensor::zeros({0, T, 2, 64}, DType::kFloat32, kCUDA0);
    ops::write_kv_quantized(none, x, x, 0);
    CHECK(ops::attention_quantized(Tensor::zeros({0, T, 6, 64}, DType::kFloat32, kCUDA0), none, 0).shape() == (std::vector<int64_t>{0, T, 6, 64}));
    CHECK(ops::read_kv_quantized(none, 8, 1).first.numel() == 0);
  }
  ops::QuantizedKV c = ops::QuantizedKV::allocate(2, 64, 1, 64, 4, kCUDA0);
  CHECK(ops::attention_quantized(Tensor::zeros({1, 0, 6, 64}, DType::kFloat32, kCUDA0), c, 64).numel() == 0);
}

}  // namespace

int main() {
  run("empty_calls", empty_calls);
  for (int bits : {4, 8}) {
    run("head_64_" + std::to_string(bits), [&] { generates(64, false, bits, 0, 0); });
    run("head_128_normed_window_" + std::to_string(bits), [&] { generates(128, true, bits, 40, 2); });
  }
  std::printf("%d cases, %d failed\n", g_cases, g_bad);
  return g_bad ? 1 : 0;
}
