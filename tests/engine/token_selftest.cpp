// Self-test of a 4-bit decoder from prompts to sampled tokens (include/ie_hip_model.hpp over
// include/ie_hip_engine.hpp). TEST INFRASTRUCTURE.
//
// The same 2-layer decoder is built twice, with 4-bit matrices (group scales that are powers of two, zero
// points) and with the BF16 matrices that those stand for, which hold every value exactly. Both run the
// same prompts and decode steps (graphs recorded, then replayed); after each the residual streams and the
// logits agree to the float32 rounding of sums taken in two orders: max |d| / max |ref| <= 1e-5. Then the
// 4-bit model's logits are adjusted and sampled on the device, and the tokens fed back: with top-k 1 the
// tokens are argmax's, under a grammar mask only its tokens appear, and a banned token does not.
//
// usage: token_selftest      exit status 0 when every check passes.
#include <cstdio>
#include <random>
#include <string>
#include <vector>

#include "ie_hip_model.hpp"
#include "oracle.h"

using namespace ie::hip;

namespace {

constexpr int kLayers = 2, H = 896, I = 1280, V = 1000, QD = 896, KVD = 128;

int g_tests = 0, g_fail = 0;
void result(bool ok, const std::string& what) {
  ++g_tests;
  if (!ok) ++g_fail;
  std::printf("%s %s\n", ok ? "ok  " : "FAIL", what.c_str());
  std::fflush(stdout);
}

/* One matrix in both formats. */
struct Both {
  std::vector<uint8_t> q, zero;
  std::vector<float> scale;
  std::vector<uint16_t> bf16;
  MatrixView q4, plain;
  Both(std::mt19937& rng, int rows, int cols, int group, float base) {
    const int groups = (cols + group - 1) / group;
    q.resize(size_t(rows) * cols / 2);
    bf16.resize(size_t(rows) * cols);
    scale.resize(size_t(rows) * groups);
    zero.resize(size_t(rows) * groups);
    for (auto& s : scale) s = base / float(1 << rng() % 2);
    for (auto& z : zero) z = uint8_t(6 + rng() % 4);
    for (int r = 0; r < rows; ++r)
      for (int c = 0; c < cols; ++c) {
        const int v = int(rng() % 16);
        const size_t g = size_t(r) * groups + c / group;
        q[(size_t(r) * cols + c) / 2] |= uint8_t(c & 1 ? v << 4 : v);
        bf16[size_t(r) * cols + c] = orc_f32_to_bf16(float(v - zero[g]) * scale[g]);
      }
    q4.data = q.data();
    q4.rows = rows;
    q4.cols = cols;
    q4.q4_group = group;
    q4.q4_scale = scale.data();
    q4.q4_scale_dtype = IE_KV_F32;
    q4.q4_zero = zero.data();
    plain.data = bf16.data();
    plain.rows = rows;
    plain.cols = cols;
  }
};

template <class T>
std::vector<T> download(const void* d, size_t n) {
  std::vector<T> h(n);
  check(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost), "download");
  return h;
}

/* Host values in device memory. */
template <class T>
struct Device {
  T* p = nullptr;
  explicit Device(const std::vector<T>& h) {
    check(hipMalloc(reinterpret_cast<void**>(&p), h.size() * sizeof(T)), "hipMalloc");
    set(h);
  }
  ~Device() { (void)hipFree(p); }
  void set(const std::vector<T>& h) {
    check(hipMemcpy(p, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice), "upload");
  }
};

}  // namespace

int main() {
  std::mt19937 rng(20261206u);
  std::normal_distribution<float> n01(0.0f, 1.0f);
  auto values = [&](size_t n, float base, float s) {
    std::vector<float> v(n);
    for (auto& e : v) e = base + s * n01(rng);
    return v;
  };
  try {
    std::vector<uint16_t> embed(size_t(V) * H);
    for (auto& e : embed) e = orc_f32_to_bf16(n01(rng));
    const std::vector<float> final_norm = values(H, 1.0f, 0.1f);
    Both head(rng, V, H, 64, 0.0625f);
    std::vector<std::vector<float>> norms, biases;
    std::vector<Both> mats;
    mats.reserve(7 * kLayers);
    ModelView q4, plain;
    for (ModelView* m : {&q4, &plain}) {
      m->embed.data = embed.data();
      m->embed.rows = V;
      m->embed.cols = H;
      m->final_norm = final_norm.data();
    }
    q4.lm_head = head.q4;
    plain.lm_head = head.plain;
    norms.reserve(2 * kLayers);
    biases.reserve(3 * kLayers);
    for (int l = 0; l < kLayers; ++l) {
      LayerView a;
      norms.push_back(values(H, 1.0f, 0.1f));
      a.input_norm = norms.back().data();
      norms.push_back(values(H, 1.0f, 0.1f));
      a.post_norm = norms.back().data();
      const float* b[3];
      for (int i = 0; i < 3; ++i) {
        biases.push_back(values(i ? KVD : QD, 0.0f, 0.1f));
        b[i] = biases.back().data();
      }
      a.bq = b[0];
      a.bk = b[1];
      a.bv = b[2];
      LayerView c = a;
      auto put = [&](MatrixView LayerView::*m, int rows, int cols, int group) {
        mats.emplace_back(rng, rows, cols, group, 0.0078125f);
        a.*m = mats.back().q4;
        c.*m = mats.back().plain;
      };
      put(&LayerView::wq, QD, H, 128);
      put(&LayerView::wk, KVD, H, 128);
      put(&LayerView::wv, KVD, H, 128);
      put(&LayerView::wo, H, QD, 32);
      put(&LayerView::w_gate, I, H, 64);
      put(&LayerView::w_up, I, H, 64);
      put(&LayerView::w_down, H, I, 128);
      q4.layers.push_back(a);
      plain.layers.push_back(c);
    }
    KvConfig cfg;
    cfg.num_layers = kLayers;
    ModelShape shape;
    shape.hidden = H;
    shape.intermediate = I;
    shape.vocab = V;
    EngineLimits lim;
    lim.max_batch = 4;
    lim.max_seq_len = 256;
    lim.num_pages = 64;
    lim.step_rows = 64;
    lim.logit_rows = 64;
    KvEngine e4(cfg, lim, IE_KV_F32, true), e16(cfg, lim, IE_KV_F32, true);
    DecoderModel m4(cfg, shape, q4, e4.limits().step_rows, e4.limits().logit_rows, 4);
    DecoderModel m16(cfg, shape, plain, e16.limits().step_rows, e16.limits().logit_rows);
    e4.set_body(m4.body(e4));
    e16.set_body(m16.body(e16));
    try {
      ModelView bad = q4;
      bad.embed = head.q4;
      DecoderModel refused(cfg, shape, bad, 4, 4);
      result(false, "a 4-bit embedding is refused");
    } catch (const std::exception&) {
      result(true, "a 4-bit embedding is refused");
    }
    auto step = [&](const std::string& what, const std::vector<int>& seq, const std::vector<int>& pos,
                    const std::vector<int32_t>& ids, bool decode) {
      const int T = int(seq.size());
      std::vector<int> all(T);
      for (int i = 0; i < T; ++i) all[i] = i;
      e4.run(seq, pos, ids, all, decode);
      e4.sync();
      e16.run(seq, pos, ids, all, decode);
      e16.sync();
      double mae = 0;
      size_t worst = 0;
      const auto x = download<float>(m4.x(), size_t(T) * H), xr = download<float>(m16.x(), size_t(T) * H);
      const auto l = download<float>(m4.logits(), size_t(T) * V);
      const auto lr = download<float>(m16.logits(), size_t(T) * V);
      const double rx = orc_compare(x.data(), xr.data(), x.size(), &mae, &worst);
      const double rl = orc_compare(l.data(), lr.data(), l.size(), &mae, &worst);
      char buf[160];
      std::snprintf(buf, sizeof(buf), "%s: residual rel %.2e, logits rel %.2e (graph %d)", what.c_str(), rx,
                    rl, int(e4.last_step().graph));
      result(rx <= 1e-5 && rl <= 1e-5, buf);
      return l;
    };
    auto ids = [&](int n) {
      std::vector<int32_t> v(n);
      for (auto& i : v) i = int32_t(rng() % V);
      return v;
    };
    const int s0 = e4.open_sequence(), s1 = e4.open_sequence();
    result(e16.open_sequence() == s0 && e16.open_sequence() == s1, "sequences");
    std::vector<int> p40(40), p17(17);
    for (int i = 0; i < 40; ++i) p40[i] = i;
    for (int i = 0; i < 17; ++i) p17[i] = i;
    step("prompt of 40", std::vector<int>(40, s0), p40, ids(40), false);
    step("prompt of 17", std::vector<int>(17, s1), p17, ids(17), false);

    // Row 0: top-k 1. Row 1: a grammar of 5 tokens, the first of them banned by a bias.
    constexpr int kWords = (V + 31) / 32;
    std::vector<uint32_t> mask(kWords, 0);
    const int allowed[5] = {3, 77, 400, 512, 999};
    for (int t : allowed) mask[t / 32] |= 1u << (t % 32);
    Device<uint32_t> d_mask(mask);
    Device<int32_t> d_mask_row({-1, 0}), d_bias_token({allowed[0]}), d_bias_start({0, 0}), d_bias_len({0, 1});
    Device<float> d_bias_value({-1e9f});
    Device<int32_t> d_history(std::vector<int32_t>(2 * 64, 0)), d_start({0, 64}), d_len({0, 0});
    Device<float> d_rep({1.3f, 1.0f}), d_pres({0.0f, 0.5f}), d_temp({0.7f, 5.0f}), d_p({1.0f, 0.99f}), d_u({0.f, 0.f});
    Device<int32_t> d_k({1, 0});
    ie_logit_rules rules{};
    rules.history = d_history.p;
    rules.history_start = d_start.p;
    rules.history_len = d_len.p;
    rules.history_size = 2 * 64;
    rules.repetition = d_rep.p;
    rules.presence = d_pres.p;
    rules.bias_token = d_bias_token.p;
    rules.bias_value = d_bias_value.p;
    rules.bias_start = d_bias_start.p;
    rules.bias_len = d_bias_len.p;
    rules.bias_size = 1;
    rules.mask = d_mask.p;
    rules.mask_row = d_mask_row.p;
    rules.mask_rows = 1;
    std::vector<int32_t> next = ids(2), history(2 * 64, 0);
    std::uniform_real_distribution<float> u01(0.0f, 1.0f);
    for (int i = 0; i < 6; ++i) {
      step("decode batch 2, step " + std::to_string(i), {s0, s1}, {40 + i, 17 + i}, next, true);
      d_history.set(history);
      d_len.set({i, i});
      d_u.set({u01(rng), u01(rng)});
      m4.adjust(2, rules, e4.stream());
      m4.argmax(1, e4.stream());
      e4.sync();
      const int32_t greedy = download<int32_t>(m4.tokens(), 1)[0];
      m4.sample(2, d_temp.p, d_k.p, d_p.p, nullptr, d_u.p, e4.stream());
      e4.sync();
      next = download<int32_t>(m4.tokens(), 2);
      bool in = false;
      for (int t = 1; t < 5; ++t) in = in || next[1] == allowed[t];
      result(next[0] == greedy && in, "tokens " + std::to_string(next[0]) + " and " + std::to_string(next[1]));
      history[i] = next[0];
      history[64 + i] = next[1];
    }
    try {
      m4.sample(5, d_temp.p, d_k.p, d_p.p, nullptr, d_u.p, e4.stream());
      result(false, "more rows than planned are refused");
    } catch (const std::exception&) {
      result(true, "more rows than planned are refused");
    }
  } catch (const std::exception& e) {
    result(false, std::string("exception: ") + e.what());
  }
  std::printf("%d checks, %d failures\n", g_tests, g_fail);
  return g_fail ? 1 : 0;
}
