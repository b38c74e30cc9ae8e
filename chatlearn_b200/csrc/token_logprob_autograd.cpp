// Differentiable form of the token statistics: a node of the autograd graph in C++, whose two kernels are in
// token_logprob.cu (a Python node costs more than the kernels where rows are few).
#include <torch/extension.h>

std::vector<at::Tensor> token_logprob_fwd(const at::Tensor& z, const at::Tensor& tokens, int64_t n, double inv_temp);
at::Tensor token_logprob_bwd(const at::Tensor& z, const at::Tensor& tokens, const at::Tensor& ent, const at::Tensor& stats,
                             const at::Tensor& ids, const c10::optional<at::Tensor>& g_lp, const c10::optional<at::Tensor>& g_ent,
                             const c10::optional<at::Tensor>& g_top, double inv_temp);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

const char* const kOnce = "token_logprobs is differentiable once";

// The gradient where a graph of it is asked for: a node that refuses to be differentiated, so that nobody takes a gradient
// that depends on the logits for a constant.
struct TokenLogprobGrad : torch::autograd::Function<TokenLogprobGrad> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& z, const at::Tensor& tokens, const at::Tensor& ent, const at::Tensor& stats,
                            const at::Tensor& ids, const c10::optional<at::Tensor>& g_lp, const c10::optional<at::Tensor>& g_ent,
                            const c10::optional<at::Tensor>& g_top, double inv_temp) {
    return token_logprob_bwd(z, tokens, ent, stats, ids, g_lp, g_ent, g_top, inv_temp);
  }
  static variable_list backward(AutogradContext*, variable_list) { TORCH_CHECK(false, kOnce); }
};

struct TokenLogprob : torch::autograd::Function<TokenLogprob> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& tokens, int64_t n, double inv_temp) {
    auto out = token_logprob_fwd(z, tokens, n, inv_temp);
    if (out.empty()) return {};
    ctx->save_for_backward({z, tokens, out[1], out[4], out[3]});
    ctx->saved_data["inv_temp"] = inv_temp;
    ctx->mark_non_differentiable({out[3]});
    ctx->set_materialize_grads(false);
    out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    auto plain = [](const at::Tensor& t) -> c10::optional<at::Tensor> {
      if (!t.defined()) return c10::nullopt;
      return t.to(at::kFloat).contiguous();
    };
    const auto lp = plain(g[0]), ent = plain(g[1]), top = plain(g[2]);
    const double inv_temp = ctx->saved_data["inv_temp"].toDouble();
    at::Tensor dz;
    if (lp || ent || top) {
      if (at::GradMode::is_enabled()) {
        dz = TokenLogprobGrad::apply(saved[0], saved[1], saved[2], saved[3], saved[4], lp, ent, top, inv_temp);
      } else {
        at::AutoDispatchBelowADInplaceOrView below;
        dz = token_logprob_bwd(saved[0], saved[1], saved[2], saved[3], saved[4], lp, ent, top, inv_temp);
      }
    }
    return {dz, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

// {log-prob, entropy, alternatives' log-probs, their ids}; empty where the arguments are not as the kernel takes them
std::vector<at::Tensor> token_logprob_apply(const at::Tensor& z, const at::Tensor& tokens, int64_t n, double inv_temp) {
  if (z._fw_grad(0).defined()) return {};          // forward mode: for the caller to refuse
  return TokenLogprob::apply(z, tokens, n, inv_temp);
}
