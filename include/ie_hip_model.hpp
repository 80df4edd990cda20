/* The decode step around the paged-KV path: a Qwen2 decoder's weights on the
 * device and its work as a KvEngine LayerBody, in C++17 over the C ABI of
 * libie_hip.so. With KvEngine this is the reference's CudaEngine forward
 * (src/cuda/cuda_runner.cu:418-470):
 *   begin               x = E[ids]                               (embedding)
 *   per layer, around the engine's RoPE + paged append + attention:
 *     before_attention  q, k, v = rmsnorm(x) . W^T + b          (one launch)
 *     after_attention   x += attn . Wo^T;
 *                       mid = silu(xn . Wg^T) * (xn . Wu^T), xn = rmsnorm(x)
 *                                                                (one launch);
 *                       x += mid . Wd^T
 *   (each rmsnorm folded into the projection after it: ie_hip_rmsnorm_qkv_proj,
 *   ie_hip_rmsnorm_gate_up_silu)
 *   end                 for the rows that want logits: xg = rmsnorm(x[rows]);
 *                       logits = xg . E_out^T
 * The rows that want logits are gathered before the final norm, which is the
 * same per row as the reference's norm-then-gather (src/cuda/cuda_runner.cu:
 * 461-464) and skips the norm of the other rows of a prompt.
 *
 * Weights arrive as a view of host memory (ModelView): BF16 bits, INT8 with one
 * f32 scale per row, or (any matrix but the embedding) 4 bits with a scale per
 * row and group of columns, in the reference's layout (nn.Linear [out, in]);
 * norms and biases f32. One device allocation holds them all; Wq, Wk and Wv are
 * stacked for the one-launch q/k/v projection. Before a 4-bit projection the
 * rmsnorm is a launch of its own. After a step, adjust() and sample() (or
 * argmax()) turn its logits into tokens on the device. Header-only. */
#ifndef IE_HIP_MODEL_HPP_
#define IE_HIP_MODEL_HPP_

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "ie_hip_engine.hpp"

namespace ie::hip {

/* The rest of the model shape (the reference's Config, src/config.h:10-26). */
struct ModelShape {
  int hidden = 896;
  int intermediate = 4864;
  int vocab = 151936;
  float rms_eps = 1e-6f;
};

/* A host matrix [rows, cols]: BF16 bits, INT8 values with a scale per row, or
 * (q4_group > 0) 4-bit values with their groups' scales and zero points, laid
 * out as an ie_matrix_q4. */
struct MatrixView {
  const void* data = nullptr;
  const float* scale = nullptr;  // INT8 only
  bool int8 = false;
  int rows = 0, cols = 0;
  int q4_group = 0;                  // columns of a group: 32, 64 or 128
  const void* q4_scale = nullptr;    // [rows, ceil(cols / group)] of q4_scale_dtype
  int q4_scale_dtype = IE_KV_F16;    // IE_KV_F32, _F16 or _BF16
  const uint8_t* q4_zero = nullptr;  // [rows, ceil(cols / group)], or null: 8
  int groups() const { return (cols + q4_group - 1) / q4_group; }
  size_t data_bytes() const {
    return q4_group > 0 ? size_t(rows) * (cols / 2) : size_t(rows) * cols * (int8 ? 1 : 2);
  }
  size_t q4_scale_bytes() const {
    return size_t(rows) * groups() * (q4_scale_dtype == IE_KV_F32 ? 4 : 2);
  }
};

/* One layer's host weights (the reference's LayerWeights, src/weights.h:22-30);
 * a null bias means the model has none. */
struct LayerView {
  const float* input_norm = nullptr;
  const float* post_norm = nullptr;
  MatrixView wq, wk, wv, wo;
  const float *bq = nullptr, *bk = nullptr, *bv = nullptr;
  MatrixView w_gate, w_up, w_down;
};

/* The model's host weights; lm_head.data == nullptr ties the LM head to the
 * embedding (Weights::lm_head_matrix, src/weights.h:38). */
struct ModelView {
  MatrixView embed, lm_head;
  const float* final_norm = nullptr;
  std::vector<LayerView> layers;
};

class DecoderModel {
 public:
  /* Uploads the weights. `rows` and `logit_rows` are the engine's step
   * capacities (EngineLimits after construction: KvEngine::limits());
   * `sample_rows` logit rows may be given to sample() (0: none, and no memory). */
  DecoderModel(const KvConfig& kv, const ModelShape& shape, const ModelView& w, int rows,
               int logit_rows, int sample_rows = 0)
      : kv_(kv), shape_(shape), rows_(rows), logit_rows_(logit_rows), sample_rows_(sample_rows) {
    const int H = shape.hidden, I = shape.intermediate, QD = kv.q_dim(), KVD = kv.kv_dim();
    if (int(w.layers.size()) != kv.num_layers)
      throw std::runtime_error("DecoderModel: layer count differs from the engine's");
    expect(w.embed, shape.vocab, H, "embedding");
    if (w.embed.q4_group > 0)
      throw std::runtime_error("DecoderModel: the embedding takes BF16 or INT8");
    if (sample_rows < 0 || sample_rows > logit_rows)
      throw std::runtime_error("DecoderModel: more rows to sample than logits");
    if (w.lm_head.data) expect(w.lm_head, shape.vocab, H, "lm_head");
    if (!w.final_norm) throw std::runtime_error("DecoderModel: no final norm");
    int8_ = w.embed.int8;

    // Sizing pass, then one allocation, then the copies.
    struct Pending {
      size_t off;
      const void* src;
      size_t bytes;
    };
    std::vector<Pending> copies;
    auto put = [&](const void* src, size_t bytes) {
      const size_t off = arena_.add<unsigned char>(bytes);
      copies.push_back({off, src, bytes});
      return off;
    };
    struct MatOff {
      size_t data = 0, scale = 0, zero = 0;
      bool int8 = false;
      int rows = 0, cols = 0, group = 0, scale_dtype = 0;
      bool has_zero = false;
    };
    size_t workspace = 0;
    auto sized = [&](MatOff& o, const MatrixView& m, int max_rows) {
      o.int8 = m.int8;
      o.rows = m.rows;
      o.cols = m.cols;
      o.group = m.q4_group;
      o.scale_dtype = m.q4_scale_dtype;
      o.has_zero = m.q4_group > 0 && m.q4_zero;
      if (m.q4_group > 0)
        workspace = std::max(workspace, matmul_q4_workspace_bytes(max_rows, m.cols));
    };
    auto put_matrix = [&](const MatrixView& m, int max_rows) {
      MatOff o;
      sized(o, m, max_rows);
      o.data = put(m.data, m.data_bytes());
      if (m.q4_group > 0) {
        o.scale = put(m.q4_scale, m.q4_scale_bytes());
        if (o.has_zero) o.zero = put(m.q4_zero, size_t(m.rows) * m.groups());
      } else if (m.int8) {
        o.scale = put(m.scale, size_t(m.rows) * sizeof(float));
      }
      return o;
    };
    // Wq, Wk, Wv stacked into one region (and their scales, and their biases).
    std::vector<std::vector<float>> zero_bias;
    auto put_stacked = [&](const LayerView& L, MatOff& m, size_t& bias, bool& has_bias) {
      // The parts of a member (bytes of Wq, Wk, Wv) one after another, in one region.
      auto stack = [&](const void* q, const void* k, const void* v, auto bytes) {
        const size_t nq = bytes(L.wq), nk = bytes(L.wk), nv = bytes(L.wv);
        const size_t at = arena_.add<unsigned char>(nq + nk + nv);
        copies.push_back({at, q, nq});
        copies.push_back({at + nq, k, nk});
        copies.push_back({at + nq + nk, v, nv});
        return at;
      };
      sized(m, L.wq, rows);
      m.rows = QD + 2 * KVD;
      m.data = stack(L.wq.data, L.wk.data, L.wv.data, [](const MatrixView& p) { return p.data_bytes(); });
      if (m.group > 0) {
        m.scale = stack(L.wq.q4_scale, L.wk.q4_scale, L.wv.q4_scale,
                        [](const MatrixView& p) { return p.q4_scale_bytes(); });
        if (m.has_zero)
          m.zero = stack(L.wq.q4_zero, L.wk.q4_zero, L.wv.q4_zero,
                         [](const MatrixView& p) { return size_t(p.rows) * p.groups(); });
      } else if (m.int8) {
        m.scale = stack(L.wq.scale, L.wk.scale, L.wv.scale,
                        [](const MatrixView& p) { return size_t(p.rows) * sizeof(float); });
      }
      has_bias = L.bq || L.bk || L.bv;
      if (has_bias) {
        bias = arena_.add<float>(m.rows);
        const float* parts[3] = {L.bq, L.bk, L.bv};
        const int lens[3] = {QD, KVD, KVD};
        size_t at = bias;
        for (int i = 0; i < 3; ++i) {
          if (!parts[i]) {  // a model with some biases: the missing ones are zero
            zero_bias.emplace_back(lens[i], 0.0f);
            parts[i] = zero_bias.back().data();
          }
          copies.push_back({at, parts[i], size_t(lens[i]) * 4});
          at += size_t(lens[i]) * 4;
        }
      }
    };

    const MatOff embed = put_matrix(w.embed, rows);
    const MatOff head = w.lm_head.data ? put_matrix(w.lm_head, logit_rows) : embed;
    const size_t final_norm = put(w.final_norm, size_t(H) * 4);
    struct LayerOff {
      size_t input_norm, post_norm, bqkv = 0;
      bool has_bias = false;
      MatOff wqkv, wo, w_gate, w_up, w_down;
    };
    std::vector<LayerOff> lo(kv.num_layers);
    for (int l = 0; l < kv.num_layers; ++l) {
      const LayerView& L = w.layers[l];
      expect(L.wq, QD, H, "wq");
      expect(L.wk, KVD, H, "wk");
      expect(L.wv, KVD, H, "wv");
      expect(L.wo, H, QD, "wo");
      expect(L.w_gate, I, H, "w_gate");
      expect(L.w_up, I, H, "w_up");
      expect(L.w_down, H, I, "w_down");
      if (!L.input_norm || !L.post_norm) throw std::runtime_error("DecoderModel: missing norm");
      auto alike = [](const MatrixView& a, const MatrixView& b) {
        return a.int8 == b.int8 && a.q4_group == b.q4_group &&
               (a.q4_group == 0 || (a.q4_scale_dtype == b.q4_scale_dtype && !a.q4_zero == !b.q4_zero));
      };
      if (!alike(L.wk, L.wq) || !alike(L.wv, L.wq))
        throw std::runtime_error("DecoderModel: q/k/v weights in different formats");
      if (L.w_gate.q4_group != L.w_up.q4_group)
        throw std::runtime_error("DecoderModel: gate and up weights in different formats");
      lo[l].input_norm = put(L.input_norm, size_t(H) * 4);
      lo[l].post_norm = put(L.post_norm, size_t(H) * 4);
      put_stacked(L, lo[l].wqkv, lo[l].bqkv, lo[l].has_bias);
      lo[l].wo = put_matrix(L.wo, rows);
      lo[l].w_gate = put_matrix(L.w_gate, rows);
      lo[l].w_up = put_matrix(L.w_up, rows);
      lo[l].w_down = put_matrix(L.w_down, rows);
    }
    // The step's activations.
    const size_t o_x = arena_.add<float>(size_t(rows) * H);
    const size_t o_xn = arena_.add<float>(size_t(rows) * H);
    const size_t o_mid = arena_.add<float>(size_t(rows) * I);
    const size_t o_xg = arena_.add<float>(size_t(logit_rows) * H);
    const size_t o_logits = arena_.add<float>(size_t(logit_rows) * shape.vocab);
    const size_t o_tokens = arena_.add<int32_t>(logit_rows);
    const size_t o_workspace = arena_.add<unsigned char>(workspace);
    const size_t o_sample = arena_.add<unsigned char>(sample_rows_workspace_bytes(sample_rows, shape.vocab));
    arena_.commit("hipMalloc(model weights)");
    for (const Pending& c : copies)
      check(hipMemcpy(arena_.at<unsigned char>(c.off), c.src, c.bytes, hipMemcpyHostToDevice),
            "hipMemcpy(weights)");

    auto mat = [&](const MatOff& o) {
      Weights d;
      if (o.group > 0)
        d.q4 = ie_matrix_q4{arena_.at<void>(o.data), arena_.at<void>(o.scale),
                            o.has_zero ? arena_.at<void>(o.zero) : nullptr, o.scale_dtype, o.group,
                            o.rows, o.cols};
      else
        d.plain = ie_matrix{arena_.at<void>(o.data), o.int8 ? arena_.at<float>(o.scale) : nullptr,
                            o.int8 ? 1 : 0, o.rows, o.cols};
      return d;
    };
    embed_ = mat(embed).plain;
    head_ = mat(head);
    final_norm_ = arena_.at<float>(final_norm);
    for (const LayerOff& o : lo) {
      Layer d;
      d.input_norm = arena_.at<float>(o.input_norm);
      d.post_norm = arena_.at<float>(o.post_norm);
      d.bqkv = o.has_bias ? arena_.at<float>(o.bqkv) : nullptr;
      d.wqkv = mat(o.wqkv);
      d.wo = mat(o.wo);
      d.w_gate = mat(o.w_gate);
      d.w_up = mat(o.w_up);
      d.w_down = mat(o.w_down);
      layers_.push_back(d);
    }
    x_ = arena_.at<float>(o_x);
    xn_ = arena_.at<float>(o_xn);
    mid_ = arena_.at<float>(o_mid);
    xg_ = arena_.at<float>(o_xg);
    logits_ = arena_.at<float>(o_logits);
    tokens_ = arena_.at<int32_t>(o_tokens);
    workspace_ = arena_.at<void>(o_workspace);
    sample_workspace_ = arena_.at<void>(o_sample);
  }
  DecoderModel(const DecoderModel&) = delete;
  DecoderModel& operator=(const DecoderModel&) = delete;

  /* The model's work in the engine's steps (the engine must outlive it). */
  LayerBody body(KvEngine& engine) {
    LayerBody b;
    b.begin = [this, &engine](int rows, hipStream_t s) {
      check_rows(rows);
      embedding(x_, engine.ids(), embed_, rows, s);
    };
    b.before_attention = [this, &engine](int l, int rows, hipStream_t s) {
      const Layer& L = layers_[l];
      if (L.wqkv.is_q4()) {
        rmsnorm(xn_, x_, L.input_norm, rows, shape_.hidden, shape_.rms_eps, s);
        qkv_proj_q4(engine.q(), engine.k(), engine.v(), xn_, L.wqkv.q4, L.bqkv, rows, kv_.q_dim(),
                    kv_.kv_dim(), workspace_, s);
      } else {
        rmsnorm_qkv_proj(engine.q(), engine.k(), engine.v(), x_, L.input_norm, shape_.rms_eps,
                         L.wqkv.plain, L.bqkv, rows, kv_.q_dim(), kv_.kv_dim(), s);
      }
    };
    b.after_attention = [this, &engine](int l, int rows, hipStream_t s) {
      const Layer& L = layers_[l];
      product(x_, engine.attn(), L.wo, rows, true, s);
      if (L.w_gate.is_q4()) {
        rmsnorm(xn_, x_, L.post_norm, rows, shape_.hidden, shape_.rms_eps, s);
        gate_up_silu_q4(mid_, xn_, L.w_gate.q4, L.w_up.q4, rows, workspace_, s);
      } else {
        rmsnorm_gate_up_silu(mid_, x_, L.post_norm, shape_.rms_eps, L.w_gate.plain, L.w_up.plain, rows,
                             s);
      }
      product(x_, mid_, L.w_down, rows, true, s);
    };
    b.end = [this, &engine](int rows, int n, hipStream_t s) {
      (void)rows;
      if (n == 0) return;
      gather_rows(xg_, x_, engine.logit_row_ids(), n, shape_.hidden, s);
      rmsnorm(xg_, xg_, final_norm_, n, shape_.hidden, shape_.rms_eps, s);
      product(logits_, xg_, head_, n, false, s);
    };
    return b;
  }

  /* The greedy token of each of the last step's n logit rows, on `s`. */
  void argmax(int n, hipStream_t s) { argmax_rows(tokens_, logits_, n, shape_.vocab, s); }

  /* The last step's n logit rows under their requests' rules, in place, on `s`. */
  void adjust(int n, const ie_logit_rules& rules, hipStream_t s) {
    adjust_logits(logits_, logits_, rules, n, shape_.vocab, s);
  }

  /* A token of each of the last step's n logit rows, into tokens(), on `s`: arguments
   * as for ie_hip_sample_rows. */
  void sample(int n, const float* temperature, const int32_t* top_k, const float* top_p,
              const float* min_p, const float* u, hipStream_t s) {
    if (n > sample_rows_) throw std::runtime_error("DecoderModel: more rows to sample than planned");
    sample_rows(tokens_, logits_, temperature, top_k, top_p, min_p, u, n, shape_.vocab,
                sample_workspace_, s);
  }

  /* The final norm of all `rows` rows into xn() (for a stage report). */
  void final_norm_all(int rows, hipStream_t s) {
    rmsnorm(xn_, x_, final_norm_, rows, shape_.hidden, shape_.rms_eps, s);
  }

  float* x() { return x_; }            // [rows, hidden] residual stream
  float* xn() { return xn_; }          // [rows, hidden] normalised rows
  float* logits() { return logits_; }  // [logit rows, vocab]
  int32_t* tokens() { return tokens_; }  // [logit rows] greedy tokens
  const ModelShape& shape() const { return shape_; }
  bool int8() const { return int8_; }
  size_t device_bytes() const { return arena_.bytes(); }

 private:
  /* A matrix in its format. */
  struct Weights {
    ie_matrix plain{};
    ie_matrix_q4 q4{};
    bool is_q4() const { return q4.data != nullptr; }
  };
  struct Layer {
    const float *input_norm, *post_norm, *bqkv;
    Weights wqkv, wo, w_gate, w_up, w_down;
  };

  void product(float* y, const float* x, const Weights& w, int rows, bool accumulate, hipStream_t s) {
    if (w.is_q4())
      matmul_q4(y, x, w.q4, nullptr, rows, accumulate, workspace_, s);
    else
      matmul(y, x, w.plain, nullptr, rows, accumulate, s);
  }

  static void expect(const MatrixView& m, int rows, int cols, const char* what) {
    if (!m.data || m.rows != rows || m.cols != cols || (m.int8 && !m.scale) || m.q4_group < 0 ||
        (m.q4_group > 0 && (m.int8 || !m.q4_scale || m.cols % 2)))
      throw std::runtime_error(std::string("DecoderModel: ") + what + " missing or of the wrong shape");
  }
  void check_rows(int rows) const {
    if (rows < 0 || rows > rows_) throw std::runtime_error("DecoderModel: more rows than the step holds");
  }

  KvConfig kv_;
  ModelShape shape_;
  int rows_, logit_rows_, sample_rows_;
  bool int8_ = false;
  DeviceArena arena_;
  ie_matrix embed_{};
  Weights head_;
  const float* final_norm_ = nullptr;
  std::vector<Layer> layers_;
  float *x_ = nullptr, *xn_ = nullptr, *mid_ = nullptr, *xg_ = nullptr, *logits_ = nullptr;
  int32_t* tokens_ = nullptr;
  void *workspace_ = nullptr, *sample_workspace_ = nullptr;
};

}  // namespace ie::hip

#endif  // IE_HIP_MODEL_HPP_
