// Autograd of the packed-sequence operators, on the host side of C++: a
// forward and backward pass of a short call costs what its launches cost,
// without the interpreter between the engine and the kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

std::vector<Tensor> attn_packed_fwd(Tensor q, Tensor k, Tensor v, Tensor cu,
                                    OptTensor lengths, bool causal,
                                    int64_t window, double scale);
std::vector<Tensor> attn_packed_bwd(Tensor q, Tensor k, Tensor v, Tensor o,
                                    Tensor dout, Tensor lse, Tensor cu,
                                    OptTensor lengths, bool causal,
                                    int64_t window, double scale);
bool attn_rows_aligned(const Tensor& t);
std::vector<Tensor> rope_axes(Tensor q, Tensor k, Tensor pos, Tensor cosb,
                              Tensor sinb, std::vector<int64_t> sections,
                              bool backward);
std::vector<Tensor> block_norm_fwd(Tensor h, Tensor x, Tensor w1, Tensor w2,
                                   OptTensor gate, double alpha, double eps,
                                   bool train);
std::vector<Tensor> block_norm_bwd(Tensor dn, Tensor ds, Tensor h, Tensor x,
                                   Tensor w1, Tensor w2, OptTensor gate,
                                   Tensor r1, Tensor r2, double alpha);

namespace {

// Allocations and views inside of a function need no trace of their own.
using Untraced = at::AutoDispatchBelowADInplaceOrView;

// Whether a call goes through its Function: for a gradient, or because an
// input carries a forward-mode tangent, which the Function refuses (also
// without grad mode, which says nothing of tangents).
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  const bool on = at::GradMode::is_enabled();
  for (const auto* t : ts)
    if (t->defined() &&
        ((on && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined()))
      return true;
  return false;
}

OptTensor maybe(const Tensor& t) {
  return t.defined() ? OptTensor(t) : c10::nullopt;
}

// Gradients that raise if they are differentiated again.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const auto& g : grads)
    in.push_back(g.defined() ? g.detach().requires_grad_() : g);
  torch::autograd::DelayedError error(
      std::string(what) + ": a second derivative is not supported",
      (int64_t)in.size());
  return error.apply(std::move(in));
}

// t, or a copy of it where 16-byte reads cannot follow its strides (an
// expanded gradient, whose strides are 0, is read as it is)
Tensor aligned_rows(const Tensor& t) {
  if (attn_rows_aligned(t)) return t;
  auto c = t.contiguous();
  return attn_rows_aligned(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}

Tensor dense_rows(const Tensor& t) {
  return t.stride(-1) == 1 ? t : t.contiguous();
}

struct PackedAttn : Function<PackedAttn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                        const Tensor& v, const Tensor& cu,
                        const OptTensor& lengths, bool causal, int64_t window,
                        double scale) {
    Untraced untraced;
    auto r = attn_packed_fwd(q, k, v, cu, lengths, causal, window, scale);
    ctx->save_for_backward({q, k, v, r[0], r[1], cu,
                            lengths.value_or(Tensor())});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    variable_list g;
    {
      Untraced untraced;
      g = attn_packed_bwd(s[0], s[1], s[2], s[3], aligned_rows(grad[0]), s[4],
                          s[5], maybe(s[6]),
                          ctx->saved_data["causal"].toBool(),
                          ctx->saved_data["window"].toInt(),
                          ctx->saved_data["scale"].toDouble());
    }
    g = once(std::move(g), "flash_attention_packed");
    return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

struct RopeAxes : Function<RopeAxes> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q,
                               const Tensor& k, const Tensor& pos,
                               const Tensor& cosb, const Tensor& sinb,
                               std::vector<int64_t> sections) {
    ctx->save_for_backward({pos, cosb, sinb});
    ctx->saved_data["sections"] = sections;
    Untraced untraced;
    return rope_axes(q, k, pos, cosb, sinb, sections, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    variable_list g;
    {
      Untraced untraced;
      g = rope_axes(dense_rows(grad[0]), dense_rows(grad[1]), s[0], s[1], s[2],
                    ctx->saved_data["sections"].toIntVector(), true);
    }
    g = once(std::move(g), "fused_rope_axes");
    return {g[0], g[1], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// The gate as [G, D]: inside of the function, where a view costs no node.
OptTensor gate_rows(const OptTensor& gate, const Tensor& h) {
  if (!gate) return gate;
  return gate->contiguous().view({gate->numel() / h.size(-1), h.size(-1)});
}

struct BlockNorm : Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& h,
                               const Tensor& x, const Tensor& w1,
                               const Tensor& w2, const OptTensor& gate,
                               double alpha, double eps) {
    Untraced untraced;
    auto r = block_norm_fwd(h, x, w1, w2, gate_rows(gate, h), alpha, eps,
                            true);
    // the sum is computed again in backward, from h and x
    ctx->save_for_backward({h, x, w1, w2, gate.value_or(Tensor()), r[2],
                            r[3]});
    ctx->saved_data["alpha"] = alpha;
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    variable_list g;
    {
      Untraced untraced;
      g = block_norm_bwd(grad[0].contiguous(), grad[1].contiguous(), s[0],
                         s[1], s[2], s[3], gate_rows(maybe(s[4]), s[0]), s[5],
                         s[6], ctx->saved_data["alpha"].toDouble());
      g[4] = s[4].defined() ? g[4].view(s[4].sizes()) : Tensor();
    }
    g = once(std::move(g), "fused_block_norm");
    return {g[0], g[1], g[2], g[3], g[4], Tensor(), Tensor()};
  }
};

}  // namespace

Tensor attn_packed(Tensor q, Tensor k, Tensor v, Tensor cu, OptTensor lengths,
                   bool causal, int64_t window, double scale) {
  q = aligned_rows(q);
  k = aligned_rows(k);
  v = aligned_rows(v);
  cu = cu.contiguous();
  if (lengths) lengths = lengths->contiguous();
  if (!wants_grad({&q, &k, &v}))
    return attn_packed_fwd(q, k, v, cu, lengths, causal, window, scale)[0];
  return PackedAttn::apply(q, k, v, cu, lengths, causal, window, scale);
}

std::vector<Tensor> rope_axes_grad(Tensor q, Tensor k, Tensor pos,
                                   Tensor cosb, Tensor sinb,
                                   std::vector<int64_t> sections) {
  q = dense_rows(q);
  k = dense_rows(k);
  pos = pos.contiguous();
  TORCH_CHECK(!cosb._fw_grad(0).defined() && !sinb._fw_grad(0).defined(),
              "fused_rope_axes: tables with a forward-mode tangent are not "
              "supported");
  cosb = cosb.detach().contiguous();
  sinb = sinb.detach().contiguous();
  if (!wants_grad({&q, &k}))
    return rope_axes(q, k, pos, cosb, sinb, sections, false);
  return RopeAxes::apply(q, k, pos, cosb, sinb, sections);
}

std::vector<Tensor> block_norm(Tensor h, Tensor x, Tensor w1, Tensor w2,
                               OptTensor gate, double alpha, double eps) {
  h = h.contiguous();
  x = x.contiguous();
  w1 = w1.contiguous();
  w2 = w2.contiguous();
  const Tensor none;
  if (!wants_grad({&h, &x, &w1, &w2, gate ? &*gate : &none})) {
    auto r = block_norm_fwd(h, x, w1, w2, gate_rows(gate, h), alpha, eps,
                            false);
    return {r[0], r[1]};
  }
  return BlockNorm::apply(h, x, w1, w2, gate, alpha, eps);
}
