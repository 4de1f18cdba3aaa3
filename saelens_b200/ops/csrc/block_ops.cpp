// The block operators as a program calls them: shapes are checked and flattened, outputs allocated,
// the kernel launched and the autograd node made in one call from Python.  A small call's time is
// the host's (a token through a norm: 24 us with these steps in Python, 9 here, of which the device
// works 2.7), so none of them is left there.
#include "block_ops.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "check.h"

namespace sb {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Opt = c10::optional<torch::Tensor>;

bool wants_grad(const torch::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const Opt& t) { return t && t->requires_grad(); }

// Forward-mode derivatives are not computed: an input's tangent is refused, not silently dropped.
bool has_tangent(const torch::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const Opt& t) { return t && has_tangent(*t); }

Opt opt(const torch::Tensor& t) { return t.defined() ? Opt(t) : Opt(); }

// [..., D] as [rows, D] with contiguous rows: a view where the layout allows it.
torch::Tensor rows_of(const torch::Tensor& t) {
  const int64_t D = t.size(-1);
  torch::Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / D, D});
  return r.stride(1) == 1 || D == 1 ? r : r.contiguous();
}

// Backward passes of one order: a second one through them is refused, not silently zero.  check_once sees
// incoming gradients that have a graph; `once` marks gradients that depend on more than those, so
// that a derivative of them, whatever the incoming ones, is an error when it is asked for.
void check_once(const variable_list& grads, const char* name) {
  if (!at::GradMode::is_enabled()) return;
  for (const auto& g : grads) SB_CHECK(!wants_grad(g), name, " is differentiable once");
}

variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined())
      g = (*std::make_shared<torch::autograd::DelayedError>(sb::detail::check_msg(name, " is differentiable once"), 1))(
          {g.detach().requires_grad_()})[0];
  return grads;
}

bool is_float(const torch::Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 || s == at::kHalf || s == at::kFloat;
}

// ------------------------------------------------------------------------------ fp8 projection
void check_status(const torch::Tensor& status, const char* where) {
  const int code = status.item<int>();
  if (code != 0) {
    status.zero_();
    SB_CHECK(false, where, ": native kernel reported status ", code);
  }
}

torch::Tensor product(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& scale, const Opt& bias,
                      bool transposed, const torch::Tensor& status) {
  const torch::Tensor x2 = rows_of(x);
  const int64_t F = weight.size(transposed ? 1 : 0);
  torch::Tensor out = torch::empty({x2.size(0), F}, x.options());
  fp8_product(x2, weight, scale, bias, transposed, out, status);
  if (x.dim() == 2) return out;
  auto shape = x.sizes().vec();
  shape.back() = F;
  return out.view(shape);
}

struct LinearFp8 : torch::autograd::Function<LinearFp8> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight,
                               const torch::Tensor& scale, const Opt& bias, const torch::Tensor& status, bool read_status) {
    ctx->save_for_backward({weight, scale});
    ctx->saved_data["status"] = status;
    ctx->saved_data["read_status"] = read_status;
    return product(x, weight, scale, bias, false, status);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once(grads, "linear_fp8");
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor status = ctx->saved_data["status"].toTensor();
    torch::Tensor dx = product(grads[0], saved[0], saved[1], {}, true, status);
    if (ctx->saved_data["read_status"].toBool()) check_status(status, "linear_fp8 (backward)");
    return {dx, {}, {}, {}, {}, {}};
  }
};

// ------------------------------------------------------------------------------ residual_norm
Opt gate_rows(const Opt& gate) {
  return !gate || gate->dim() == 2 ? gate : Opt(gate->view({gate->numel() / gate->size(-1), gate->size(-1)}));
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& branch,
                               const torch::Tensor& w, const Opt& b, const Opt& post_w, const Opt& post_b, const Opt& gate,
                               int64_t div, int64_t mode, double eps, double post_eps, double scale, bool layer,
                               bool one_plus, bool round_branch) {
    // shapes change inside the node: a view for each input and output would be nodes of their own
    const torch::Tensor x2 = rows_of(x), b2 = rows_of(branch);
    torch::Tensor stream = torch::empty(x.sizes(), x.options()), normed = torch::empty(x.sizes(), x.options());
    torch::Tensor stats = torch::empty({4, x2.size(0)}, x.options().dtype(at::kFloat));
    residual_norm_fwd(x2, b2, w, b, post_w, post_b, gate_rows(gate), div, eps, post_eps, scale, layer, one_plus, round_branch,
                      rows_of(stream), rows_of(normed), stats);
    auto or_none = [](const Opt& t) { return t ? *t : torch::Tensor(); };
    // the branch is read again only where its own values enter a gradient
    ctx->save_for_backward({stream, post_w || gate ? b2 : torch::Tensor(), w, or_none(post_w), or_none(post_b), or_none(gate), stats});
    ctx->saved_data["args"] = c10::ivalue::Tuple::create({div, mode, scale, layer, one_plus});
    ctx->saved_data["has"] = c10::ivalue::Tuple::create({b.has_value(), post_w.has_value(), post_b.has_value(), gate.has_value()});
    ctx->set_materialize_grads(false);
    return {stream, normed};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once(grads, "residual_norm");
    variable_list out(15);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const torch::Tensor &stream = s[0], &w = s[2];
    const auto& args = ctx->saved_data["args"].toTupleRef().elements();
    const auto& has = ctx->saved_data["has"].toTupleRef().elements();
    const int64_t div = args[0].toInt(), mode = args[1].toInt();
    const double scale = args[2].toDouble();
    // A gradient may be a view that starts anywhere (a slice of what a concatenation got).  Rows too wide for
    // single values, which the forward pass took by 16-byte vectors, are copied then.
    auto rows = [](const torch::Tensor& t) {
      if (!t.defined()) return Opt();
      const torch::Tensor r = rows_of(t);
      return Opt(residual_norm_needs_vectors(r.size(1)) && !residual_norm_vectors(r) ? r.clone(at::MemoryFormat::Contiguous) : r);
    };
    // needs_input_grad counts the tensors that were given
    size_t edge = 3;
    auto next_needed = [&](int i) { return has[i].toBool() && ctx->needs_input_grad(edge++); };
    auto like = [&](bool needed, const torch::Tensor& t) { return needed ? Opt(torch::empty(t.sizes(), t.options())) : Opt(); };
    // with nothing between the branch and the stream their gradients are one
    const bool alike = !s[3].defined() && !s[5].defined() && scale == 1.0;
    torch::Tensor dx = torch::empty(stream.sizes(), stream.options());
    const Opt dbranch = like(!alike && ctx->needs_input_grad(1), stream), dw = like(ctx->needs_input_grad(2), w);
    const Opt db = like(next_needed(0), w), dpw = like(next_needed(1), s[3]), dpb = like(next_needed(2), s[4]);
    const Opt dg = like(next_needed(3), s[5]);
    const torch::Tensor s2 = rows_of(stream);
    residual_norm_bwd(rows(grads[0]), rows(grads[1]), s2, s[1].defined() ? s[1] : s2, w, opt(s[3]), opt(s[4]),
                      gate_rows(opt(s[5])), div, mode, scale, args[3].toBool(), args[4].toBool(), s[6], rows_of(dx),
                      dbranch ? Opt(rows_of(*dbranch)) : dbranch, dw, db, dpw, dpb, gate_rows(dg));
    if (ctx->needs_input_grad(0)) out[0] = dx;
    if (ctx->needs_input_grad(1)) out[1] = alike ? dx : *dbranch;
    if (dw) out[2] = *dw;
    if (db) out[3] = *db;
    if (dpw) out[4] = *dpw;
    if (dpb) out[5] = *dpb;
    if (dg) out[6] = *dg;
    return once(std::move(out), "residual_norm");
  }
};

// ------------------------------------------------------------------------------ rotary
torch::Tensor last_contiguous(const torch::Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// Whether no value of t is there twice: from the least stride on, each dimension steps over all that the
// ones before it span.  So it is in what slices, transposes and views leave of a whole tensor; other
// layouts that hold each value once are rare, and refused with the rest.
bool apart(const torch::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return true;
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  }
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;
  for (const auto& [stride, size] : dims) {
    if (stride < span) return false;
    span += (size - 1) * stride;
  }
  return true;
}

// Whether q and k of one storage may hold a value in common.  Views of one tensor have the same strides
// between sequences and tokens: they are apart if what they span of a sequence or of a token is, or if
// their heads interleave with one stride and never meet.  Others are apart if all they span is.
bool may_share(const torch::Tensor& q, const torch::Tensor& k) {
  if (q.numel() == 0 || k.numel() == 0 || q.storage().data_ptr().get() != k.storage().data_ptr().get()) return false;
  const int64_t d = q.size(3), oq = q.storage_offset(), ok = k.storage_offset();
  auto span = [](const torch::Tensor& t, int from) {
    int64_t n = 1;
    for (int i = from; i < 4; ++i) n += (t.size(i) - 1) * t.stride(i);
    return n;
  };
  if (oq + span(q, 0) <= ok || ok + span(k, 0) <= oq) return false;
  for (int i = 0; i < 2; ++i) {
    // what one entry of dimension i spans; it must not reach into the next one's for this to say anything
    const int64_t eq = oq + span(q, i + 1), ek = ok + span(k, i + 1);
    if (q.size(i) > 1 && (q.stride(i) != k.stride(i) || std::max(eq, ek) - std::min(oq, ok) > q.stride(i))) return true;
    if (eq <= ok || ek <= oq) return false;
  }
  const int64_t step = q.size(2) > 1 ? q.stride(2) : k.stride(2);
  if ((q.size(2) > 1 && k.size(2) > 1 && q.stride(2) != k.stride(2)) || step < 2 * d) return true;
  const int64_t apart = ((ok - oq) % step + step) % step;
  return apart < d || apart > step - d;
}

// What is written in place counts as a change: autograd then notices where it had saved the old values.
// (Tensors made in inference mode count nothing.)
void changed(const torch::Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

std::tuple<torch::Tensor, torch::Tensor> turn(const torch::Tensor& q0, const torch::Tensor& k0, const torch::Tensor& freq,
                                              const Opt& pos, int64_t offset, bool interleaved, bool inverse, double factor) {
  const torch::Tensor q = last_contiguous(q0);
  torch::Tensor qo = torch::empty(q.sizes(), q.options()), ko;
  if (!k0.defined()) {
    rotary_fwd(q, {}, freq, pos, offset, interleaved, inverse, factor, qo, {});
  } else {
    const torch::Tensor k = last_contiguous(k0);
    ko = torch::empty(k.sizes(), k.options());
    rotary_fwd(q, k, freq, pos, offset, interleaved, inverse, factor, qo, ko);
  }
  return {qo, ko};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& q, const Opt& k, const torch::Tensor& freq,
                               const Opt& pos, int64_t offset, bool interleaved, bool inverse, double factor) {
    ctx->save_for_backward({freq, pos ? *pos : torch::Tensor()});
    ctx->saved_data["args"] = c10::ivalue::Tuple::create({offset, interleaved, inverse, factor, k.has_value()});
    ctx->set_materialize_grads(false);
    auto [qo, ko] = turn(q, k ? *k : torch::Tensor(), freq, pos, offset, interleaved, inverse, factor);
    if (!k) return {qo};
    return {qo, ko};
  }
  // the transposed rotation, differentiable in its turn
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto& a = ctx->saved_data["args"].toTupleRef().elements();
    const torch::Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : torch::Tensor();
    variable_list out(8);
    const torch::Tensor& first = dq.defined() ? dq : dk;
    if (!first.defined()) return out;
    const Opt second = dq.defined() && dk.defined() ? Opt(dk) : Opt();
    variable_list r;
    const int64_t offset = a[0].toInt();
    const bool interleaved = a[1].toBool(), inverse = !a[2].toBool();
    const double factor = a[3].toDouble();
    if (at::GradMode::is_enabled() && (wants_grad(first) || wants_grad(second))) {
      r = Rotary::apply(first, second, s[0], opt(s[1]), offset, interleaved, inverse, factor);
    } else {
      auto [x, y] = turn(first, second ? *second : torch::Tensor(), s[0], opt(s[1]), offset, interleaved, inverse, factor);
      r = {x, y};
    }
    if (dq.defined()) {
      out[0] = r[0];
      if (dk.defined()) out[1] = r[1];
    } else {
      out[1] = r[0];
    }
    return out;
  }
};

}  // namespace

// x [..., K] times the frozen e4m3 weight [N, K] (scales [N / 128, K / 128]) plus bias: [..., N] in
// x's type; differentiable in x.  read_status: the backward pass reads the status word itself.
torch::Tensor linear_fp8(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& scale, const Opt& bias,
                         const torch::Tensor& status, bool read_status) {
  SB_VALUE(x.dim() >= 1 && is_float(x) && x.size(-1) >= 1, "linear_fp8: x must be bf16, fp16 or fp32 [..., width]");
  SB_VALUE(weight.dim() == 2 && weight.scalar_type() == at::kFloat8_e4m3fn && weight.size(0) >= 1 && weight.size(1) == x.size(-1),
           "linear_fp8: the weight must be float8_e4m3fn [features, ", x.size(-1), "]");
  SB_VALUE(!has_tangent(x) && !has_tangent(scale) && !has_tangent(bias), "linear_fp8 has no forward-mode derivative");
  if (at::GradMode::is_enabled()) {
    SB_VALUE(!scale.requires_grad() && !wants_grad(bias) && !weight.requires_grad(),
             "linear_fp8: the weight, its scales and the bias are frozen; only x has a gradient");
    if (x.requires_grad()) return LinearFp8::apply(x, weight, scale, bias, status, read_status);
  }
  return product(x, weight, scale, bias, false, status);
}

std::tuple<torch::Tensor, torch::Tensor> residual_norm(const torch::Tensor& x, const torch::Tensor& branch,
                                                       const torch::Tensor& w, const Opt& b, bool layer, double eps,
                                                       bool one_plus, const Opt& post_w, const Opt& post_b,
                                                       double post_eps, const Opt& gate, double scale, bool round_branch) {
  SB_VALUE(x.dim() >= 1 && is_float(x) && x.size(-1) >= 1, "residual_norm: x must be bf16, fp16 or fp32 [..., D]");
  SB_VALUE(branch.sizes() == x.sizes(), "residual_norm: branch must have x's shape");
  const int64_t D = x.size(-1);
  auto check = [&](const torch::Tensor& t, const char* name, bool vector) {
    SB_VALUE(t.scalar_type() == x.scalar_type() && t.device() == x.device(), "residual_norm: ", name, " must be of x's type on x's device");
    SB_VALUE(!vector || (t.dim() == 1 && t.size(0) == D), "residual_norm: ", name, " must be [", D, "]");
  };
  SB_VALUE(layer || (!b && !post_b), "residual_norm: RMS norms have no bias");
  SB_VALUE(post_w || !post_b, "residual_norm: post_bias without post_weight");
  check(branch, "branch", false);
  check(w, "weight", true);
  if (b) check(*b, "bias", true);
  if (post_w) check(*post_w, "post_weight", true);
  if (post_b) check(*post_b, "post_bias", true);
  SB_VALUE(!has_tangent(x) && !has_tangent(branch) && !has_tangent(w) && !has_tangent(b) && !has_tangent(post_w) &&
               !has_tangent(post_b) && !has_tangent(gate),
           "residual_norm has no forward-mode derivative");
  auto vector = [](const Opt& t) { return t && !t->is_contiguous() ? Opt(t->contiguous()) : t; };
  const torch::Tensor wc = w.is_contiguous() ? w : w.contiguous();
  const Opt bc = vector(b), pw = vector(post_w), pb = vector(post_b);
  // the gate: one row for all rows (1), one for several consecutive ones (2) or one each (3)
  Opt g;
  int64_t div = 1, mode = 0;
  if (gate) {
    check(*gate, "gate", false);
    const int64_t lead = x.dim() - 1, own = gate->dim() - 1;
    SB_VALUE(own >= 0 && own <= lead && gate->size(-1) == D, "residual_norm: gate does not match x");
    int64_t last = -1;
    for (int64_t i = 0; i < own; ++i)
      if (gate->size(i) != 1) last = lead - own + i;
    for (int64_t i = 0; i <= last; ++i)
      SB_VALUE((i < lead - own ? 1 : gate->size(i - (lead - own))) == x.size(i),
               "residual_norm: gate must be one row for all of x or one for each entry of its leading dimensions");
    for (int64_t i = last + 1; i < lead; ++i) div *= x.size(i);
    mode = last < 0 ? 1 : div == 1 ? 3 : 2;
    div = std::max<int64_t>(div, 1);
    g = gate->is_contiguous() ? *gate : gate->contiguous();
  }
  const int vectors = int(wants_grad(w)) + int(wants_grad(b)) + int(wants_grad(post_w)) + int(wants_grad(post_b));
  if (at::GradMode::is_enabled() && (x.requires_grad() || branch.requires_grad() || vectors || wants_grad(gate))) {
    const int sums = vectors + int(wants_grad(gate) && mode != 3);
    SB_VALUE(residual_norm_bwd_fits(D, sums), "residual_norm: ", sums, " column sums of width ", D, " do not fit the backward pass");
    auto r = ResidualNorm::apply(x, branch, wc, bc, pw, pb, g, div, mode, eps, post_eps, scale, layer, one_plus, round_branch);
    return {r[0], r[1]};
  }
  const torch::Tensor x2 = rows_of(x), b2 = rows_of(branch);
  torch::Tensor stream = torch::empty(x2.sizes(), x.options()), normed = torch::empty(x2.sizes(), x.options());
  residual_norm_fwd(x2, b2, wc, bc, pw, pb, gate_rows(g), div, eps, post_eps, scale, layer, one_plus, round_branch, stream, normed, {});
  if (x.dim() == 2) return {stream, normed};
  return {stream.view(x.sizes()), normed.view(x.sizes())};
}

// q and k (or q alone) turned; see rotary.cu.
std::tuple<torch::Tensor, Opt> rotary(const torch::Tensor& q, const Opt& k, const torch::Tensor& freq, const Opt& positions,
                                      int64_t offset, bool interleaved, double factor, bool inplace) {
  SB_VALUE(q.dim() == 4 && is_float(q), "rotary: q must be bf16, fp16 or fp32 [B, S, H, d]");
  const int64_t B = q.size(0), S = q.size(1), d = q.size(3);
  SB_VALUE(!k || (k->dim() == 4 && k->scalar_type() == q.scalar_type() && k->device() == q.device() && k->size(0) == B &&
                  k->size(1) == S && k->size(3) == d),
           "rotary: k does not match q");
  SB_VALUE(freq.dim() == 1 && freq.scalar_type() == at::kDouble && !freq.requires_grad() && freq.numel() >= 1 && 2 * freq.numel() <= d,
           "rotary: freq must be constant fp64 [rot / 2] with rot from 2 to ", d);
  SB_VALUE(!has_tangent(q) && !has_tangent(k) && !has_tangent(freq), "rotary has no forward-mode derivative");
  Opt pos;
  if (positions) {
    const auto t = positions->scalar_type();
    SB_VALUE((t == at::kLong || t == at::kInt) && positions->dim() <= 2, "rotary: positions must be int64 or int32 [B, S]");
    SB_VALUE(offset == 0, "rotary: either positions or an offset");
    bool fits = true;
    for (int64_t i = 0; i < positions->dim(); ++i) {
      const int64_t n = positions->size(positions->dim() - 1 - i), want = i == 0 ? S : B;
      fits = fits && (n == want || n == 1);
    }
    SB_VALUE(fits, "rotary: positions do not broadcast to [", B, ", ", S, "]");
    pos = positions->expand({B, S});
  }
  SB_VALUE(freq.device() == q.device() && (!pos || pos->device() == q.device()), "rotary: all tensors must be on one CUDA device");
  const torch::Tensor f = freq.is_contiguous() ? freq : freq.contiguous();
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k));
  if (inplace) {
    SB_VALUE(!grad, "rotary: not in place where gradients are wanted");
    auto check = [&](const torch::Tensor& t) {
      SB_VALUE((d <= 1 || t.stride(3) == 1) && apart(t), "rotary: in place needs contiguous channels and no value twice");
    };
    check(q);
    if (k) {
      check(*k);
      SB_VALUE(!may_share(q, *k), "rotary: in place, q and k must not share values");
    }
    rotary_fwd(q, k, f, pos, offset, interleaved, false, factor, q, k);
    changed(q);
    if (k) changed(*k);
    return {q, k};
  }
  if (grad) {
    auto r = Rotary::apply(q, k, f, pos, offset, interleaved, false, factor);
    return {r[0], k ? Opt(r[1]) : Opt()};
  }
  auto [qo, ko] = turn(q, k ? *k : torch::Tensor(), f, pos, offset, interleaved, false, factor);
  return {qo, opt(ko)};
}

}  // namespace sb
