// Autograd nodes of the block operators, so that a call and its backward stay out of the interpreter:
// at a few thousand elements an operator costs what its launch costs, and a Python node adds some 30 us
// to a forward and backward.  The Python layer keeps its own nodes for what belongs to the sharding engine
// (gradients that go into its fp32 buffers) and for the CPU path; both call the same kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <cstdio>

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

Tensor qk_norm_rope_fwd(Tensor x, Tensor wq, Tensor wk, Tensor cos_t, Tensor sin_t, c10::optional<Tensor> pos,
                        int64_t nq, int64_t nkv, int64_t hd, int64_t seqlen, double eps);
Tensor qk_norm_rope_bwd(Tensor g, Tensor x, Tensor wq, Tensor wk, Tensor cos_t, Tensor sin_t,
                        c10::optional<Tensor> pos, int64_t nq, int64_t nkv, int64_t hd, int64_t seqlen, double eps,
                        Tensor dwq, Tensor dwk, bool accumulate);
Tensor dropout_add(Tensor x, c10::optional<Tensor> residual, int64_t cut, int64_t seed, int64_t start);
std::vector<Tensor> token_logprobs_fwd(Tensor x, Tensor tokens, double temperature, int64_t top_k, int64_t ignore,
                                       bool want_state);
void token_logprobs_bwd(Tensor x, Tensor tokens, Tensor state, c10::optional<Tensor> g_lp, c10::optional<Tensor> g_ent,
                        double temperature, Tensor dx);
std::vector<Tensor> fp8_quantize_with_tiles(Tensor x, Tensor s, int64_t rows);
std::vector<Tensor> fp8_quantize(Tensor x, bool square, bool plain, bool transposed);
std::vector<Tensor> fp8_quantize_tiles(Tensor x, bool square, bool plain, bool transposed);
void fp8_gemm(Tensor A, Tensor tA, Tensor B, Tensor tB, Tensor D, c10::optional<Tensor> R, bool accumulate);
void fp8_product(Tensor A, Tensor sA, c10::optional<Tensor> tA, Tensor B, Tensor sB, c10::optional<Tensor> tB, Tensor D,
                 c10::optional<Tensor> R, bool accumulate);

Tensor dropout_add_autograd(Tensor x, c10::optional<Tensor> residual, int64_t cut, int64_t seed, int64_t start);

// A kernel's result has no graph: under create_graph a term through it would count as constant and be missing
// from the second derivative without a word.  This lets the gradient g of the running node through and makes a
// differentiation of it raise, for all that the node (or the gradients dys it was given) depends on.
Tensor first_order(Tensor g, const std::string& op, const std::vector<Tensor>& dys) {
  if (!g.defined() || !at::GradMode::is_enabled()) return g;
  torch::autograd::edge_list edges;
  if (const auto node = torch::autograd::get_current_node())
    for (const auto& e : node->next_edges())
      if (e.is_valid()) edges.push_back(e);
  for (const Tensor& dy : dys)
    if (dy.defined() && dy.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(dy));
  g = g.detach();
  torch::autograd::set_history(g, std::make_shared<torch::autograd::Error>(op + " has no second derivative", std::move(edges)));
  return g;
}

namespace {

struct QkNormRope : public Function<QkNormRope> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wq, const Tensor& wk, const Tensor& cos_t,
                        const Tensor& sin_t, const c10::optional<Tensor>& pos, int64_t nq, int64_t nkv, int64_t hd,
                        int64_t seqlen, double eps) {
    ctx->save_for_backward({x, wq, wk, cos_t, sin_t, pos.value_or(Tensor())});
    ctx->saved_data["c"] = std::vector<int64_t>{nq, nkv, hd, seqlen};
    ctx->saved_data["eps"] = eps;
    return qk_norm_rope_fwd(x, wq, wk, cos_t, sin_t, pos, nq, nkv, hd, seqlen, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto c = ctx->saved_data["c"].toIntVector();
    Tensor g = grads[0];
    if (g.stride(1) != 1) g = g.contiguous();
    Tensor dwq = torch::empty_like(s[1]), dwk = torch::empty_like(s[2]);
    Tensor dx = qk_norm_rope_bwd(g, s[0], s[1], s[2], s[3], s[4],
                                 s[5].defined() ? c10::optional<Tensor>(s[5]) : c10::nullopt, c[0], c[1], c[2], c[3],
                                 ctx->saved_data["eps"].toDouble(), dwq, dwk, false);
    const char* op = "qk_norm_rope";
    return {first_order(dx, op, grads), first_order(dwq, op, grads), first_order(dwk, op, grads), {}, {}, {}, {}, {}, {}, {}, {}};
  }
};

struct DropoutAdd : public Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& residual, int64_t cut,
                        int64_t seed, int64_t start) {
    ctx->saved_data["c"] = std::vector<int64_t>{cut, seed, start, residual.has_value()};
    return dropout_add(x, residual, cut, seed, start);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto c = ctx->saved_data["c"].toIntVector();
    Tensor dx;
    // (linear in the gradient: the same node again where the gradient is to be differentiated)
    if (ctx->needs_input_grad(0)) dx = dropout_add_autograd(grads[0].contiguous(), c10::nullopt, c[0], c[1], c[2]);
    // an input that was not given takes no gradient
    return {dx, c[3] ? grads[0] : Tensor(), {}, {}, {}};
  }
};

Tensor row_grad(const Tensor& g) { return g.defined() ? g.to(at::kFloat).contiguous() : g; }

struct TokenLogProbs : public Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& tokens, double temperature,
                               int64_t top_k, int64_t ignore) {
    auto r = token_logprobs_fwd(x, tokens, temperature, top_k, ignore, true);
    ctx->save_for_backward({x, tokens, r.back()});
    r.pop_back();
    ctx->saved_data["t"] = temperature;
    if (top_k > 0) ctx->mark_non_differentiable({r[2], r[3]});
    ctx->set_materialize_grads(false);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor& x = s[0];
    // the gradient's rows lie as the logits' rows do (padded vocabulary buffers included)
    const int64_t M = x.size(0), V = x.size(1);
    int64_t pitch = M > 1 ? std::max(x.stride(0), V) : V;
    if (pitch > 2 * V + 1024) pitch = V;
    Tensor dx = torch::empty({M, pitch}, x.options());
    if (pitch != V) dx = dx.narrow(1, 0, V);
    const Tensor gl = row_grad(grads[0]), ge = row_grad(grads[1]);  // (of the tokens' shape)
    token_logprobs_bwd(x, s[1], s[2], gl.defined() ? c10::optional<Tensor>(gl) : c10::nullopt,
                       ge.defined() ? c10::optional<Tensor>(ge) : c10::nullopt, ctx->saved_data["t"].toDouble(), dx);
    return {first_order(dx, "token_log_probs", grads), {}, {}, {}, {}};
  }
};

struct LinearFp8 : public Function<LinearFp8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const c10::optional<Tensor>& residual) {
    const bool need_x = x.requires_grad(), need_w = w.requires_grad();
    auto xq = fp8_quantize_tiles(x, false, true, need_w);  // codes, scale tiles; of the transpose: 2, 3
    auto wq = fp8_quantize_tiles(w, true, true, need_x);
    Tensor y = torch::empty({x.size(0), w.size(0)}, x.options());
    fp8_gemm(xq[0], xq[1], wq[0], wq[1], y, residual, false);
    ctx->save_for_backward({xq[2], xq[3], wq[2], wq[3]});
    ctx->saved_data["t"] = w.scalar_type();
    ctx->saved_data["r"] = residual.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    Tensor dx, dw;
    if (need_x || need_w) {
      Tensor g = grads[0].contiguous();
      auto gq = fp8_quantize_tiles(g, false, need_x, need_w);
      if (need_x) {
        dx = torch::empty({g.size(0), s[2].size(0)}, g.options());
        fp8_gemm(gq[0], gq[1], s[2], s[3], dx, c10::nullopt, false);
      }
      if (need_w) {
        const auto t = ctx->saved_data["t"].toScalarType();
        dw = torch::empty({g.size(1), s[0].size(0)}, g.options().dtype(t == at::kHalf ? at::kFloat : t));
        fp8_gemm(gq[2], gq[3], s[0], s[1], dw, c10::nullopt, false);
        dw = dw.to(t);
      }
    }
    return {first_order(dx, "linear_fp8", grads), first_order(dw, "linear_fp8", grads), ctx->saved_data["r"].toBool() ? grads[0] : Tensor()};
  }
};

}  // namespace

// A call that nothing will differentiate skips the node.  A tangent (forward mode, which works without grad mode)
// goes to the node, which refuses it.
static bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
static bool tracked(const Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || has_tangent(t); }

Tensor qk_norm_rope_autograd(Tensor x, Tensor wq, Tensor wk, Tensor cos_t, Tensor sin_t, c10::optional<Tensor> pos,
                             int64_t nq, int64_t nkv, int64_t hd, int64_t seqlen, double eps) {
  if (!tracked(x) && !tracked(wq) && !tracked(wk)) return qk_norm_rope_fwd(x, wq, wk, cos_t, sin_t, pos, nq, nkv, hd, seqlen, eps);
  return QkNormRope::apply(x, wq, wk, cos_t, sin_t, pos, nq, nkv, hd, seqlen, eps);
}
Tensor dropout_add_autograd(Tensor x, c10::optional<Tensor> residual, int64_t cut, int64_t seed, int64_t start) {
  if (!tracked(x) && !(residual.has_value() && tracked(*residual))) return dropout_add(x, residual, cut, seed, start);
  return DropoutAdd::apply(x, residual, cut, seed, start);
}
// logits [..., V], tokens [...] -> {logprob, entropy} or {logprob, entropy, top log probabilities, top tokens}
std::vector<Tensor> token_logprobs_autograd(Tensor x, Tensor tokens, double temperature, int64_t top_k, int64_t ignore) {
  if (x.dim() != 2) x = x.reshape({-1, x.size(-1)});
  if (x.stride(1) != 1 && x.numel() > 0) x = x.contiguous();
  if (!tokens.is_contiguous()) tokens = tokens.contiguous();
  if (!tracked(x)) return token_logprobs_fwd(x, tokens, temperature, top_k, ignore, false);
  return TokenLogProbs::apply(x, tokens, temperature, top_k, ignore);
}
// x [T, K] bf16, w [N, K], residual [T, N] bf16 or none
Tensor linear_fp8_autograd(Tensor x, Tensor w, c10::optional<Tensor> residual) {
  if (!tracked(x) && !tracked(w) && !(residual.has_value() && tracked(*residual))) {
    // no backward: codes as they lie alone (8192 x 4096: 24 us instead of 34)
    auto xq = fp8_quantize_tiles(x, false, true, false), wq = fp8_quantize_tiles(w, true, true, false);
    Tensor y = torch::empty({x.size(0), w.size(0)}, x.options());
    fp8_gemm(xq[0], xq[1], wq[0], wq[1], y, residual, false);
    return y;
  }
  return LinearFp8::apply(x, w, residual);
}

// ValueError unless q is e4m3 [rows, cols] and s its e8m0 scales in 1 x 128 or 128 x 128 blocks.
void fp8_check_blocks(const Tensor& q, const Tensor& s) {
  char msg[160];
  if (q.dim() != 2 || q.scalar_type() != at::kFloat8_e4m3fn || s.scalar_type() != at::kFloat8_e8m0fnu) {
    std::snprintf(msg, sizeof(msg), "8-bit blocks are e4m3 [rows, cols] codes with e8m0 scales, got %s and %s",
                  c10::toString(q.scalar_type()), c10::toString(s.scalar_type()));
    TORCH_CHECK_VALUE(false, msg);
  }
  const long rows = q.size(0), cols = q.size(1), blocks = (rows + 127) / 128;
  const long sr = s.dim() > 0 ? s.size(0) : 0, sc = s.dim() > 1 ? s.size(1) : 0;
  if (s.dim() == 2 && (sr == blocks || sr == rows) && sc == (cols + 127) / 128) return;
  std::snprintf(msg, sizeof(msg), "scales [%ld, %ld] fit neither 1 x 128 nor 128 x 128 blocks of %ld x %ld", sr, sc, rows, cols);
  TORCH_CHECK_VALUE(false, msg);
}

// x [T, K] bf16 with weights kept in 8 bits: values [N, K] e4m3, scales e8m0, their tiles or none
Tensor linear_fp8_kept(Tensor x, Tensor values, Tensor scales, c10::optional<Tensor> tiles,
                       c10::optional<Tensor> residual) {
  fp8_check_blocks(values, scales);
  TORCH_CHECK(!has_tangent(x) && !(residual.has_value() && has_tangent(*residual)),
              "weights kept in 8 bits have no derivative: call linear_fp8 with the weight tensor");
  auto xq = tiles.has_value() ? fp8_quantize(x, false, true, false) : fp8_quantize_with_tiles(x, scales, values.size(0));
  Tensor y = torch::empty({x.size(0), values.size(0)}, x.options());
  fp8_product(xq[0], xq[1], xq[2], values, scales, tiles.has_value() ? tiles : xq[3], y, residual, false);
  return y;
}
