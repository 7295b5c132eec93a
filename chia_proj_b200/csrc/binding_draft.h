// binding_draft.h -- the Python side of include/chia_draft.h and chia_rope.h.
#pragma once
#include "binding_args.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

decltype(&chia_tree_tables) g_tree_tables;
decltype(&chia_tree_attn) g_tree_attn;
decltype(&chia_verify_drafts) g_verify;
decltype(&chia_cache_compact) g_compact;
decltype(&chia_qk_norm_rope) g_rope;
decltype(&chia_qk_norm_rope_bwd) g_rope_bwd;
decltype(&chia_qk_norm_rope_bwd_workspace_bytes) g_rope_bytes;

int any_type(const Tensor &t) { return t.scalar_type() == at::kFloat ? CHIA_DTYPE_F32 : value_type(t); }

// The offsets of requests: int32 [B + 1], B > 0.
const Tensor &offsets(const Args &a, int i, const at::Device &dev) {
  const Tensor &cu = a.tensor(i, "cu_q", 1);
  if (cu.size(0) < 2) throw ValueError("cu_q must have an entry more than there are requests, two at least");
  return a.ints(i, "cu_q", {cu.size(0)}, dev);
}

// ---------------------------------------------------------------------- tables
// parents, cu_q, seq_lens, status
PyObject *tree_tables(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Args a(args, nargs, 4);
    const Tensor &parents = a.tensor(0, "parents", 1);
    const at::Device dev = parents.device();
    const int64_t T = parents.size(0);
    a.ints(0, "parents", {T}, dev);
    const Tensor &cu = offsets(a, 1, dev), &lens = a.ints(2, "seq_lens", {cu.size(0) - 1}, dev);
    const c10::cuda::CUDAGuard guard(dev);
    Tensor words = at::empty({T}, parents.options().dtype(at::kLong)), positions = at::empty({T}, parents.options());
    chia_tree_params_t p{};
    p.abi_version = CHIA_DRAFT_ABI_VERSION;
    p.batch = cu.size(0) - 1;
    p.tokens = T;
    p.parents = ptr<int32_t>(parents);
    p.cu_q = ptr<int32_t>(cu);
    p.seq_lens = ptr<int32_t>(lens);
    p.positions = ptr<int32_t>(positions);
    p.ancestors = ptr<uint64_t>(words);
    p.status = reinterpret_cast<int32_t *>(a.integer(3));
    const int code = g_tree_tables(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (code != CHIA_OK) return PyLong_FromLong(code);
    return Py_BuildValue("(NN)", THPVariable_Wrap(positions), THPVariable_Wrap(words));
  });
}

// ---------------------------------------------------------------- verification
// target_probs, tokens, parents, cu_q, uniforms, draft_probs, max_tokens, status
PyObject *verify(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Args a(args, nargs, 8);
    const Tensor &probs = a.tensor(0, "target_probs", 2);
    const at::Device dev = probs.device();
    const int64_t T = probs.size(0), V = probs.size(1), most = a.integer(6);
    const int dt = any_type(probs);
    if (dt < 0) throw ValueError(std::string("dtype ") + c10::toString(probs.scalar_type()) + " unsupported (fp32, bf16 or fp16)");
    if (V < 1) throw ValueError("target_probs of an empty vocabulary");
    if (most < 1) throw ValueError("max_tokens must be >= 1");
    const Tensor &tokens = a.ints(1, "tokens", {T}, dev), &parents = a.ints(2, "parents", {T}, dev);
    const Tensor &cu = offsets(a, 3, dev);
    const Tensor &u = a.tensor(4, "uniforms", 1);
    if (u.scalar_type() != at::kFloat || u.size(0) != T || u.device() != dev || !u.is_contiguous())
      throw ValueError("uniforms must be contiguous fp32 (" + std::to_string(T) + ",) on " + dev.str());
    auto rows = [&](const Tensor &t) {  // rows that do not overlap, or that are all one
      return t.stride(1) == 1 || V == 1 ? t.stride(0) >= V || T == 1 : false;
    };
    Tensor p2 = rows(probs) ? probs : probs.contiguous(), q2;
    no_tangent(probs, "target_probs");
    if (!a.none(5)) {
      const Tensor &q = a.tensor(5, "draft_probs", 2);
      if (q.sizes() != probs.sizes() || q.scalar_type() != probs.scalar_type() || q.device() != dev)
        throw ValueError("draft_probs must match target_probs in shape, dtype and device");
      no_tangent(q, "draft_probs");
      q2 = rows(q) ? q : q.contiguous();
    }
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t B = cu.size(0) - 1;
    // one allocation for all outputs
    Tensor buf = at::empty({B + 2 * B * most}, cu.options());
    int32_t *o = ptr<int32_t>(buf);
    chia_verify_params_t p{};
    p.abi_version = CHIA_DRAFT_ABI_VERSION;
    p.dtype = dt;
    p.batch = B;
    p.tokens = T;
    p.vocab = V;
    p.max_tokens = most;
    p.target_probs = p2.data_ptr();
    p.target_stride = T > 1 ? p2.stride(0) : V;
    if (q2.defined()) {
      p.draft_probs = q2.data_ptr();
      p.draft_stride = T > 1 ? q2.stride(0) : V;
    }
    p.node_tokens = ptr<int32_t>(tokens);
    p.parents = ptr<int32_t>(parents);
    p.cu_q = ptr<int32_t>(cu);
    p.uniforms = ptr<float>(u);
    p.counts = o;
    p.out_tokens = o + B;
    p.path = o + B + B * most;
    p.status = reinterpret_cast<int32_t *>(a.integer(7));
    const int code = g_verify(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (code != CHIA_OK) return PyLong_FromLong(code);
    auto table = [&](int64_t at) {
      Tensor t = piece(buf, at, B * most);
      t.unsafeGetTensorImpl()->set_sizes_contiguous({B, most});
      return THPVariable_Wrap(t);
    };
    return Py_BuildValue("(NNN)", THPVariable_Wrap(piece(buf, 0, B)), table(B), table(B + B * most));
  });
}

// ------------------------------------------------------------------ compaction
// path, counts, cu_q, seq_lens, block_table, k_cache, v_cache, k_scale, v_scale, status, slots
PyObject *compact(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Args a(args, nargs, 11);
    const Cache c(a, 5);
    const Tensor &path = a.tensor(0, "path", 2), &table = a.tensor(4, "block_table", 2);
    const int64_t B = table.size(0), W = table.size(1), most = path.size(1);
    if (B < 1 || W < 1 || most < 1) throw ValueError("empty path or block_table");
    a.ints(0, "path", {B, most}, c.dev);
    if (!path.is_contiguous()) throw ValueError("path must be contiguous");
    a.ints(4, "block_table", {B, W}, c.dev);
    if (B > 1 && table.stride(0) < W) throw ValueError("the rows of block_table must not overlap");
    const Tensor &counts = a.ints(1, "counts", {B}, c.dev), &cu = a.ints(2, "cu_q", {B + 1}, c.dev);
    const Tensor &lens = a.ints(3, "seq_lens", {B}, c.dev);
    const c10::cuda::CUDAGuard guard(c.dev);
    Tensor keep = at::empty({B}, lens.options());
    chia_compact_params_t p{};
    p.abi_version = CHIA_COMPACT_ABI_VERSION;
    p.cache_dtype = c.type;
    p.head_dim = static_cast<int32_t>(c.dim);
    p.heads_kv = static_cast<int32_t>(c.heads);
    p.page_size = static_cast<int32_t>(c.page);
    p.batch = B;
    p.max_tokens = most;
    p.num_pages = c.pages;
    p.table_width = W;
    p.table_stride = table.stride(0) > W ? table.stride(0) : W;
    p.path = ptr<int32_t>(path);
    p.counts = ptr<int32_t>(counts);
    p.cu_q = ptr<int32_t>(cu);
    p.seq_lens = ptr<int32_t>(lens);
    p.block_table = ptr<int32_t>(table);
    p.k_cache = c.k.data_ptr();
    p.v_cache = c.v.data_ptr();
    p.k_scale = ptr<float>(c.ks);
    p.v_scale = ptr<float>(c.vs);
    p.keep_lens = ptr<int32_t>(keep);
    p.status = reinterpret_cast<int32_t *>(a.integer(9));
    if (!a.none(10)) {
      p.tokens = a.tensor(10, "slots", 1).size(0);
      p.slots = ptr<int32_t>(a.ints(10, "slots", {p.tokens}, c.dev));
    }
    const int code = g_compact(&p, c10::cuda::getCurrentCUDAStream(c.dev.index()).stream());
    if (code != CHIA_OK) return PyLong_FromLong(code);
    for (const Tensor *t : {&c.k, &c.v, &c.ks, &c.vs}) written(*t);
    return THPVariable_Wrap(keep);
  });
}

// -------------------------------------------------------------- norm, rotation
// Queries and keys as [batch, heads, tokens, channels]: from [T, H, D], or as they are.
struct Rows {
  Tensor t;
  int64_t b, h, s, d;
  int64_t st[3];  // batch, head, token
};
bool rows_fit(const Tensor &t) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.stride(i) % 8 != 0 || t.stride(i) < 0) return false;
  return true;
}
Rows rows_of(const Tensor &t) {
  Rows r{t, 1, 0, 0, 0, {0, 0, 0}};
  if (t.dim() == 3) {
    r.s = t.size(0), r.h = t.size(1), r.d = t.size(2);
    r.st[1] = t.stride(1), r.st[2] = t.stride(0);
  } else {
    r.b = t.size(0), r.h = t.size(1), r.s = t.size(2), r.d = t.size(3);
    r.st[0] = t.stride(0), r.st[1] = t.stride(1), r.st[2] = t.stride(2);
  }
  return r;
}
// An input: a copy where its rows are not 16-byte aligned with unit stride.
Rows rows_in(const Tensor &t) { return rows_of(rows_fit(t) ? t : fitting(t)); }
// A new tensor like an input, in its order of dimensions.
Rows rows_out(const Tensor &like) {
  Tensor o = at::empty_like(like, like.options().requires_grad(false));
  if (!rows_fit(o)) o = at::empty(like.sizes(), like.options().requires_grad(false));
  return rows_of(o);
}

// The arguments of qk_norm_rope; weights and positions may be undefined.
struct RopeIn {
  Tensor q, k, qw, kw, freqs, pos;
  double eps, offset;
  bool inter;
  RopeIn() = default;
  // q, k, q_weight, k_weight, freqs, positions, eps, interleaved, weight_offset
  RopeIn(const Args &a, int i) {
    q = input(a, i, "q"), k = input(a, i + 1, "k");
    if (!a.none(i + 2)) qw = a.tensor(i + 2, "q_weight", 1);
    if (!a.none(i + 3)) kw = a.tensor(i + 3, "k_weight", 1);
    freqs = a.tensor(i + 4, "freqs", 1);
    if (!a.none(i + 5)) {
      if (!THPVariable_Check(a.v[i + 5])) throw ValueError("positions must be a tensor");
      const int64_t dim = THPVariable_Unpack(a.v[i + 5]).dim();
      const bool each = q.dim() == 4 && dim == 2;  // of each batch entry
      const int64_t shape[2] = {q.size(0), q.size(q.dim() == 3 ? 0 : 2)};
      pos = a.ints(i + 5, "positions", each ? at::IntArrayRef(shape, 2) : at::IntArrayRef(shape + 1, 1), q.device());
    }
    eps = a.number(i + 6);
    const int x = PyObject_IsTrue(a.v[i + 7]);
    if (x < 0) throw 0;
    inter = x;
    offset = a.number(i + 8);
  }
  static const Tensor &input(const Args &a, int i, const char *name) {
    if (!THPVariable_Check(a.v[i]) || (THPVariable_Unpack(a.v[i]).dim() != 3 && THPVariable_Unpack(a.v[i]).dim() != 4))
      throw ValueError(std::string(name) + " must be a 3-D or 4-D tensor");
    return a.tensor(i, name, THPVariable_Unpack(a.v[i]).dim());
  }
};

// The same checked, as the library takes it.
struct Rope {
  Rows q, k;
  Tensor qw, kw;
  chia_rope_params_t p{};
  explicit Rope(const RopeIn &in) : q(rows_in(in.q)), k(rows_in(in.k)) {
    const Tensor &qt = q.t, &kt = k.t;
    const at::Device dev = qt.device();
    const int dt = any_type(qt);
    no_tangent(in.q, "q"), no_tangent(in.k, "k");
    if (dt < 0) throw ValueError(std::string("dtype ") + c10::toString(qt.scalar_type()) + " unsupported (bf16, fp16 or fp32)");
    if (kt.scalar_type() != qt.scalar_type() || kt.device() != dev || kt.dim() != qt.dim() || k.b != q.b || k.s != q.s || k.d != q.d)
      throw ValueError("q " + str(qt.sizes()) + ", k " + str(kt.sizes()) + " must match in all but the heads, in dtype and in device");
    if (q.d != 64 && q.d != 128) throw ValueError("head_dim " + std::to_string(q.d) + " unsupported (64 or 128)");
    if (q.h < 1 || k.h < 1 || q.b < 1) throw ValueError("empty q or k");
    qw = weight(in.qw, "q_weight"), kw = weight(in.kw, "k_weight");
    if (qw.defined() && kw.defined() && qw.scalar_type() != kw.scalar_type())
      throw ValueError("q_weight, k_weight must share a dtype");
    if (in.freqs.scalar_type() != at::kLong || in.freqs.device() != dev || !in.freqs.is_contiguous())
      throw ValueError("freqs must be contiguous int64 on " + dev.str() + " (rope_frequencies makes them)");
    const int64_t rot = 2 * in.freqs.size(0);
    if (rot > q.d || rot % 8 != 0)
      throw ValueError("freqs for " + std::to_string(rot) + " channels: a multiple of 8 up to " + std::to_string(q.d));
    if (in.pos.defined()) {
      p.positions = ptr<int32_t>(in.pos);
      if (in.pos.dim() == 2) p.position_stride = in.pos.stride(0);
    }
    p.abi_version = CHIA_ROPE_ABI_VERSION;
    p.dtype = dt;
    p.weight_dtype = qw.defined() ? any_type(qw) : kw.defined() ? any_type(kw) : CHIA_DTYPE_F32;
    p.head_dim = static_cast<int32_t>(q.d);
    p.heads = static_cast<int32_t>(q.h);
    p.heads_kv = static_cast<int32_t>(k.h);
    p.rot = static_cast<int32_t>(rot);
    p.batch = q.b;
    p.seqlen = q.s;
    p.q = qt.data_ptr();
    p.k = kt.data_ptr();
    for (int x = 0; x < 3; ++x) p.q_stride[x] = q.st[x], p.k_stride[x] = k.st[x];
    if (qw.defined()) p.q_weight = qw.data_ptr();
    if (kw.defined()) p.k_weight = kw.data_ptr();
    p.freqs = ptr<uint64_t>(in.freqs);
    p.eps = static_cast<float>(in.eps);
    p.interleaved = in.inter;
    p.weight_offset = static_cast<float>(in.offset);
    if (!(p.eps >= 0.f) || !std::isfinite(p.eps) || !std::isfinite(p.weight_offset))
      throw ValueError("eps must be >= 0, eps and weight_offset finite");
  }
  Tensor weight(const Tensor &w, const char *name) const {
    if (!w.defined()) return w;
    if (w.size(0) != q.d || any_type(w) < 0 || w.device() != q.t.device())
      throw ValueError(std::string(name) + " must be bf16, fp16 or fp32 (" + std::to_string(q.d) + ",) on " + q.t.device().str() +
                       ", got " + c10::toString(w.scalar_type()) + " " + str(w.sizes()) + " on " + w.device().str());
    no_tangent(w, name);
    return w.is_contiguous() && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0
               ? w
               : w.detach().clone(at::MemoryFormat::Contiguous);
  }
  void *stream() const { return c10::cuda::getCurrentCUDAStream(q.t.device().index()).stream(); }
};

// Outputs in out; a status.
int rope_forward(const RopeIn &in, Tensor (&out)[2]) {
  Rope r(in);
  const c10::cuda::CUDAGuard guard(r.q.t.device());
  const Rows qo = rows_out(r.q.t), ko = rows_out(r.k.t);
  r.p.q_out = qo.t.data_ptr(), r.p.k_out = ko.t.data_ptr();
  for (int x = 0; x < 3; ++x) r.p.q_out_stride[x] = qo.st[x], r.p.k_out_stride[x] = ko.st[x];
  out[0] = qo.t, out[1] = ko.t;
  return g_rope(&r.p, r.stream());
}

// dq, dk, dq_weight, dk_weight (undefined where it is not wanted) in out; a status.
int rope_backward(const RopeIn &in, const Tensor &dq_out, const Tensor &dk_out, bool want_qw, bool want_kw, Tensor (&out)[4]) {
  Rope r(in);
  const Tensor *dy[2] = {&dq_out, &dk_out};
  const Rows *x[2] = {&r.q, &r.k};
  Rows g[2];
  for (int i = 0; i < 2; ++i) {
    no_tangent(*dy[i], i ? "dk_out" : "dq_out");
    if (dy[i]->sizes() != x[i]->t.sizes() || dy[i]->scalar_type() != x[i]->t.scalar_type() ||
        dy[i]->device() != r.q.t.device())
      throw ValueError(std::string(i ? "dk_out" : "dq_out") + " must match " + (i ? "k" : "q") + " in shape, dtype and device");
    g[i] = rows_in(*dy[i]);
  }
  const c10::cuda::CUDAGuard guard(r.q.t.device());
  const Rows dq = rows_out(r.q.t), dk = rows_out(r.k.t);
  for (int i = 0; i < 3; ++i) r.p.q_out_stride[i] = dq.st[i], r.p.k_out_stride[i] = dk.st[i];
  chia_rope_grads_t gr{};
  gr.dq_out = g[0].t.data_ptr(), gr.dk_out = g[1].t.data_ptr();
  for (int i = 0; i < 3; ++i) gr.dq_out_stride[i] = g[0].st[i], gr.dk_out_stride[i] = g[1].st[i];
  gr.dq = dq.t.data_ptr(), gr.dk = dk.t.data_ptr();
  out[0] = dq.t, out[1] = dk.t;
  if (r.qw.defined() && want_qw) out[2] = at::empty({r.q.d}, r.qw.options().requires_grad(false)), gr.dq_weight = out[2].data_ptr();
  if (r.kw.defined() && want_kw) out[3] = at::empty({r.q.d}, r.kw.options().requires_grad(false)), gr.dk_weight = out[3].data_ptr();
  Tensor ws;
  int64_t bytes = 0;
  if (r.qw.defined() || r.kw.defined()) {
    bytes = g_rope_bytes(&r.p);
    if (bytes < 0) throw ValueError("invalid backward parameters");
    ws = at::empty({bytes}, r.q.t.options().dtype(at::kByte).requires_grad(false));
  }
  return g_rope_bwd(&r.p, &gr, ws.defined() ? ws.data_ptr() : nullptr, bytes, r.stream());
}

PyObject *wrap(const Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }

struct Status {  // other than CHIA_OK, on its way to the function that returns it
  int code;
};

// The graph's node of a call: its inputs are kept, the backward kernel computes the norms again. (As a
// Python function of autograd's a step took 40 us of the host's time more.)
struct RopeNode : torch::autograd::Function<RopeNode> {
  using List = torch::autograd::variable_list;
  using Context = torch::autograd::AutogradContext;
  using Maybe = std::optional<Tensor>;  // (a weight that is not there has no edge)
  static List forward(Context *ctx, const Tensor &q, const Tensor &k, const Maybe &, const Maybe &, const RopeIn *in) {
    const at::AutoDispatchBelowADInplaceOrView plain;
    Tensor out[2];
    const int code = rope_forward(*in, out);
    if (code != CHIA_OK) throw Status{code};
    ctx->save_for_backward({q, k, in->qw, in->kw, in->freqs, in->pos});
    ctx->saved_data["eps"] = in->eps;
    ctx->saved_data["offset"] = in->offset;
    ctx->saved_data["inter"] = in->inter;
    return {out[0], out[1]};
  }
  static List backward(Context *ctx, List grads) {
    const List saved = ctx->get_saved_variables();
    RopeIn in;
    in.q = saved[0], in.k = saved[1], in.qw = saved[2], in.kw = saved[3], in.freqs = saved[4], in.pos = saved[5];
    in.eps = ctx->saved_data["eps"].toDouble(), in.offset = ctx->saved_data["offset"].toDouble();
    in.inter = ctx->saved_data["inter"].toBool();
    Tensor out[4];
    {
      const at::AutoDispatchBelowADInplaceOrView plain;
      const Tensor dq = grads[0].defined() ? grads[0] : at::zeros_like(in.q);
      const Tensor dk = grads[1].defined() ? grads[1] : at::zeros_like(in.k);
      size_t edge = 2;
      const bool want_qw = in.qw.defined() && ctx->needs_input_grad(edge++);
      const bool want_kw = in.kw.defined() && ctx->needs_input_grad(edge);
      const int code = rope_backward(in, dq, dk, want_qw, want_kw, out);
      if (code != CHIA_OK) throw std::runtime_error("chia_qk_norm_rope_bwd: status " + std::to_string(code));
    }
    List result = {out[0], out[1], out[2], out[3], Tensor()};
    if (c10::GradMode::is_enabled()) {
      // The gradients' own gradients are refused when they are asked for: each gets a node that throws, with
      // edges to all that the gradients depend on, so that whatever leads to one of them leads through it.
      List all;
      for (int i = 0; i < 4; ++i) all.push_back(out[i].defined() ? out[i].detach() : Tensor());
      for (const Tensor &t : {in.q, in.k, in.qw, in.kw, grads[0], grads[1]}) all.push_back(t);
      all = torch::autograd::DelayedError("qk_norm_rope has no second derivative", static_cast<int>(all.size())).apply(std::move(all));
      for (int i = 0; i < 4; ++i)
        if (out[i].defined()) result[i] = all[i];
    }
    return result;
  }
};

// the nine arguments of RopeIn
PyObject *qk_norm_rope(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const Args a(args, nargs, 9);
    const RopeIn in(a, 0);
    Tensor out[2];
    auto learns = [](const Tensor &t) { return t.defined() && t.requires_grad(); };
    if (c10::GradMode::is_enabled() && (learns(in.q) || learns(in.k) || learns(in.qw) || learns(in.kw))) {
      auto maybe = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      try {
        const auto r = RopeNode::apply(in.q, in.k, maybe(in.qw), maybe(in.kw), &in);
        out[0] = r[0], out[1] = r[1];
      } catch (const Status &s) {
        return PyLong_FromLong(s.code);
      }
    } else {
      const at::AutoDispatchBelowADInplaceOrView plain;
      const int code = rope_forward(in, out);
      if (code != CHIA_OK) return PyLong_FromLong(code);
    }
    return Py_BuildValue("(NN)", wrap(out[0]), wrap(out[1]));
  });
}

// dq_out, dk_out, then the nine arguments of RopeIn, want_q_weight, want_k_weight
PyObject *qk_norm_rope_bwd(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Args a(args, nargs, 13);
    const Tensor &dq = RopeIn::input(a, 0, "dq_out"), &dk = RopeIn::input(a, 1, "dk_out");
    const RopeIn in(a, 2);
    Tensor out[4];
    const int code = rope_backward(in, dq, dk, PyObject_IsTrue(a.v[11]), PyObject_IsTrue(a.v[12]), out);
    if (code != CHIA_OK) return PyLong_FromLong(code);
    return Py_BuildValue("(NNNN)", wrap(out[0]), wrap(out[1]), wrap(out[2]), wrap(out[3]));
  });
}

}  // namespace
