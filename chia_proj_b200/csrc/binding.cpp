// binding.cpp -- the Python side of include/chia_paged.h: argument checks, output
// tensors and workspaces of the paged 8-bit K/V cache's operators. (Those of drafted
// tokens, and of the norm and rotation of queries and keys, are in binding_draft.h.)
//
// A decode step calls these once a layer, and on an idle GPU a call is a dozen
// microseconds, so the checks are made here, on the tensors themselves: the
// same checks in Python took 9 to 15 us a call. The functions take positional
// arguments only; the public signatures and their documentation are in
// chia_proj_b200/paged.py, draft.py and rope.py, the computation in libchia_attn.so, whose entry
// points bind() is given. A status other than CHIA_OK is returned as an int.
#include "binding_args.h"
#include "binding_draft.h"

namespace {

decltype(&chia_page_tables) g_tables, g_release, g_trim;
decltype(&chia_cache_append) g_append;
decltype(&chia_paged_attn) g_attn;
decltype(&chia_paged_attn_workspace_bytes) g_bytes;

// --------------------------------------------------------------------- tables
// seq_lens, lens, block_table, free_pages, free_state, page_size, max_tokens (-1: release, -2: trim), status
PyObject *tables(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;  // outputs carry no gradients
    const Args a(args, nargs, 8);
    const Tensor &lens = a.tensor(0, "seq_lens", 1);
    const at::Device dev = lens.device();
    const int64_t B = lens.size(0), page = a.integer(5), most = a.integer(6);
    const bool release = most < 0;
    check_page(page);
    const Tensor &table = a.tensor(2, "block_table", 2), &ring = a.tensor(3, "free_pages", 1);
    if (B < 1 || table.size(1) < 1 || ring.size(0) < 1)
      throw ValueError("empty seq_lens, block_table or free_pages");
    a.ints(0, "seq_lens", {B}, dev);
    const Tensor &what = a.ints(1, most == -1 ? "done" : release ? "keep_lens" : "new_lens", {B}, dev);
    a.ints(2, "block_table", {B, table.size(1)}, dev);
    a.ints(3, "free_pages", {ring.size(0)}, dev);
    const Tensor &state = a.ints(4, "free_state", {2}, dev);
    if (B > 1 && table.stride(0) < table.size(1)) throw ValueError("the rows of block_table must not overlap");
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t T = release ? 0 : most;
    // one allocation for all outputs
    Tensor buf = at::empty({2 * T + 2 * B + 3}, lens.options());
    int32_t *o = ptr<int32_t>(buf);
    chia_tables_params_t p{};
    p.abi_version = CHIA_PAGED_ABI_VERSION;
    p.page_size = static_cast<int32_t>(page);
    p.batch = B;
    p.table_width = table.size(1);
    p.table_stride = table.stride(0) > table.size(1) ? table.stride(0) : table.size(1);
    p.ring_size = ring.size(0);
    p.max_tokens = T;
    p.seq_lens = ptr<int32_t>(lens);
    p.new_lens = ptr<int32_t>(what);
    p.block_table = ptr<int32_t>(table);
    p.free_pages = ptr<int32_t>(ring);
    p.free_state = ptr<int32_t>(state);
    p.slots = o;
    p.positions = o + T;
    p.cu_q = o + 2 * T;
    p.new_seq_lens = o + 2 * T + B + 1;
    p.new_free_state = o + 2 * T + 2 * B + 1;
    p.status = reinterpret_cast<int32_t *>(a.integer(7));
    void *stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const int code = (most == -1 ? g_release : release ? g_trim : g_tables)(&p, stream);
    if (code != CHIA_OK) return PyLong_FromLong(code);
    written(release ? ring : table);
    const int64_t at[5] = {0, T, 2 * T, 2 * T + B + 1, 2 * T + 2 * B + 1}, n[5] = {T, T, B + 1, B, 2};
    PyObject *out = PyTuple_New(release ? 2 : 5);
    for (int i = release ? 3 : 0, j = 0; i < 5; ++i, ++j)
      PyTuple_SET_ITEM(out, j, THPVariable_Wrap(piece(buf, at[i], n[i])));
    return out;
  });
}

// --------------------------------------------------------------------- append
// k, v, slots, k_cache, v_cache, k_scale, v_scale, status
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;  // outputs carry no gradients
    const Args a(args, nargs, 8);
    const Cache c(a, 3);
    const Tensor *k = &a.tensor(0, "k", 3), *v = &a.tensor(1, "v", 3);
    const int64_t T = k->size(0), shape[3] = {T, c.heads, c.dim};
    const int dt = value_type(*k);
    if (dt < 0 || v->scalar_type() != k->scalar_type())
      throw ValueError(std::string("k, v must share a type, bf16 or fp16; got ") +
                       c10::toString(k->scalar_type()) + ", " + c10::toString(v->scalar_type()));
    if (k->sizes() != at::IntArrayRef(shape, 3) || v->sizes() != k->sizes() || k->device() != c.dev ||
        v->device() != c.dev)
      throw ValueError("k, v must be " + str({shape, 3}) + " on " + c.dev.str() + ", got " + str(k->sizes()) + ", " +
                       str(v->sizes()));
    const Tensor &slots = a.ints(2, "slots", {T}, c.dev);
    no_tangent(*k, "k"), no_tangent(*v, "v");
    if (T == 0) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(c.dev);
    Tensor kc, vc;
    if (!fits(*k)) kc = fitting(*k), k = &kc;
    if (!fits(*v)) vc = fitting(*v), v = &vc;
    chia_append_params_t p{};
    p.abi_version = CHIA_PAGED_ABI_VERSION;
    p.dtype = dt;
    p.cache_dtype = c.type;
    p.head_dim = static_cast<int32_t>(c.dim);
    p.heads_kv = static_cast<int32_t>(c.heads);
    p.page_size = static_cast<int32_t>(c.page);
    p.tokens = T;
    p.num_pages = c.pages;
    p.k = k->data_ptr();
    p.v = v->data_ptr();
    p.k_stride[0] = k->stride(0), p.k_stride[1] = k->stride(1);
    p.v_stride[0] = v->stride(0), p.v_stride[1] = v->stride(1);
    p.slots = ptr<int32_t>(slots);
    p.k_cache = c.k.data_ptr();
    p.v_cache = c.v.data_ptr();
    p.k_scale = ptr<float>(c.ks);
    p.v_scale = ptr<float>(c.vs);
    p.status = reinterpret_cast<int32_t *>(a.integer(7));
    const int code = g_append(&p, c10::cuda::getCurrentCUDAStream(c.dev.index()).stream());
    if (code != CHIA_OK) return PyLong_FromLong(code);
    for (const Tensor *t : {&c.k, &c.v, &c.ks, &c.vs}) written(*t);
    Py_RETURN_NONE;
  });
}

// ------------------------------------------------------------------ attention
// Workspace of one (device, stream): as large as any call needs, zero-filled
// once. A call that a CUDA graph captures gets one of its own, zero-filled
// within the graph: the graph may be replayed beside calls on the stream that
// captured it. (The map is never freed: at exit the CUDA context may be gone.)
Tensor workspace(const at::Device &dev, void *stream) {
  static auto *held = new std::map<std::pair<int, void *>, Tensor>;
  const bool capturing =
      c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  const auto key = std::make_pair(static_cast<int>(dev.index()), stream);
  const auto it = held->find(key);
  if (it != held->end() && !capturing) return it->second;
  int64_t n = 0;
  for (int q : {16, 1024}) {  // few and many rows a K/V head, the larger head size
    chia_paged_params_t p{};
    p.abi_version = CHIA_PAGED_ABI_VERSION;
    p.head_dim = 128;
    p.heads = p.heads_kv = 1;
    p.page_size = 16;
    p.max_q = q;
    p.batch = p.tokens = p.num_pages = p.table_width = p.table_stride = 1;
    void *some = reinterpret_cast<void *>(256);
    p.q = p.o = p.workspace = some;
    p.k_cache = p.v_cache = some;
    p.k_scale = p.v_scale = static_cast<float *>(some);
    p.block_table = p.seq_lens = static_cast<int32_t *>(some);
    p.scale = 1.f;
    p.dilation = 1;
    n = std::max(n, g_bytes(&p));
  }
  if (n <= 0) throw std::runtime_error("no workspace size");
  Tensor t = at::zeros({n}, at::TensorOptions().dtype(at::kByte).device(dev));
  if (!capturing) (*held)[key] = t;
  return t;
}

// q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_q, max_q (0: not known), norm, mod, mask (tuple
// of 5), scale (None: 1 / sqrt(D)), softcap, head_param, sig_bias, out_scale, out, return_lse, wait_limit_ns, status,
// tree (None, or a tuple: positions, ancestors)
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Args a(args, nargs, 22);
    const Cache c(a, 1);
    const Tensor *q = &a.tensor(0, "q", 3);
    const int64_t T = q->size(0), H = q->size(1), D = q->size(2);
    const int dt = value_type(*q);
    if (dt < 0) throw ValueError(std::string("dtype ") + c10::toString(q->scalar_type()) + " unsupported (bf16 or fp16)");
    if (D != c.dim || H < 1 || H % c.heads != 0 || q->device() != c.dev)
      throw ValueError("q " + str(q->sizes()) + " on " + q->device().str() + " does not fit a cache " +
                       str(c.k.sizes()) + " on " + c.dev.str());
    if (q->requires_grad() && c10::GradMode::is_enabled())
      throw ValueError("paged_attention has no backward pass");
    no_tangent(*q, "q");
    const Tensor &table = a.tensor(5, "block_table", 2);
    const int64_t B = table.size(0), W = table.size(1);
    if (B < 1 || W < 1) throw ValueError("empty block_table");
    a.ints(5, "block_table", {B, W}, c.dev);
    const Tensor &lens = a.ints(6, "seq_lens", {B}, c.dev);
    if (B > 1 && table.stride(0) < W) throw ValueError("the rows of block_table must not overlap");
    const Tensor *cu = nullptr;
    if (!a.none(7))
      cu = &a.ints(7, "cu_q", {B + 1}, c.dev);
    else if (T % B != 0)
      throw ValueError(std::to_string(T) + " queries for " + std::to_string(B) + " requests need cu_q");
    const int32_t *tree_pos = nullptr;
    const uint64_t *tree_word = nullptr;
    if (!a.none(21)) {
      if (!PyTuple_Check(a.v[21]) || PyTuple_GET_SIZE(a.v[21]) != 2)
        throw ValueError("tree must be what tree_tables returns");
      const Args tree(&PyTuple_GET_ITEM(a.v[21], 0), 2, 2);
      tree_pos = ptr<int32_t>(tree.ints(0, "tree.positions", {T}, c.dev));
      const Tensor &w = tree.tensor(1, "tree.ancestors", 1);
      if (w.scalar_type() != at::kLong || w.size(0) != T || w.device() != c.dev || !w.is_contiguous())
        throw ValueError("tree.ancestors must be contiguous int64 (" + std::to_string(T) + ",) on " + c.dev.str());
      tree_word = ptr<uint64_t>(w);
    }
    int64_t max_q = a.none(8) ? (cu == nullptr ? T / B : T - B + 1) : a.integer(8);
    if (!a.none(8) && max_q < 1) throw ValueError("max_q must be >= 1");
    max_q = std::max<int64_t>(1, std::min(max_q, T));
    const c10::cuda::CUDAGuard guard(c.dev);
    Tensor qc;
    if (!fits(*q)) qc = fitting(*q), q = &qc;
    chia_paged_params_t p{};
    Tensor out, hp, lse;
    if (a.none(17)) {
      out = at::empty({T, H, D}, q->options().requires_grad(false));
    } else {
      out = a.tensor(17, "out", 3);
      if (out.sizes() != q->sizes() || out.scalar_type() != q->scalar_type() || out.device() != c.dev)
        throw ValueError("out must match q in shape, dtype and device");
      if (!fits(out)) throw ValueError("out must have unit last stride and 16-byte aligned rows");
      if (!apart(out)) throw ValueError("out must not overlap itself");
    }
    if (!a.none(14)) {
      if (!THPVariable_Check(a.v[14])) throw ValueError("head_param must be a tensor");
      hp = THPVariable_Unpack(a.v[14]);
      if (hp.numel() != H)
        throw ValueError("per-head parameter must have " + std::to_string(H) + " entries, got " +
                         std::to_string(hp.numel()));
      if (hp.scalar_type() != at::kFloat || hp.device() != c.dev || !hp.is_contiguous())
        hp = hp.detach().to(c.dev, at::kFloat).contiguous();
      p.head_param = ptr<float>(hp);
    }
    if (PyObject_IsTrue(a.v[18])) {
      lse = at::empty({T, H}, lens.options().dtype(at::kFloat));
      p.lse = ptr<float>(lse);
    }
    if (T > 0) {
      void *stream = c10::cuda::getCurrentCUDAStream(c.dev.index()).stream();
      const Tensor ws = workspace(c.dev, stream);
      p.abi_version = CHIA_PAGED_ABI_VERSION;
      p.dtype = dt;
      p.cache_dtype = c.type;
      p.head_dim = static_cast<int32_t>(D);
      p.norm = static_cast<int32_t>(a.integer(9));
      p.mod = static_cast<int32_t>(a.integer(10));
      p.heads = static_cast<int32_t>(H);
      p.heads_kv = static_cast<int32_t>(c.heads);
      p.page_size = static_cast<int32_t>(c.page);
      p.max_q = static_cast<int32_t>(max_q);
      p.batch = B;
      p.tokens = T;
      p.num_pages = c.pages;
      p.table_width = W;
      p.table_stride = table.stride(0) > W ? table.stride(0) : W;
      p.q = q->data_ptr();
      p.o = out.data_ptr();
      p.q_stride[0] = q->stride(0), p.q_stride[1] = q->stride(1);
      p.o_stride[0] = out.stride(0), p.o_stride[1] = out.stride(1);
      p.k_cache = c.k.data_ptr();
      p.v_cache = c.v.data_ptr();
      p.k_scale = ptr<float>(c.ks);
      p.v_scale = ptr<float>(c.vs);
      p.block_table = ptr<int32_t>(table);
      p.seq_lens = ptr<int32_t>(lens);
      p.cu_q = cu != nullptr ? ptr<int32_t>(*cu) : nullptr;
      p.scale = static_cast<float>(a.none(12) ? 1.0 / std::sqrt(static_cast<double>(D)) : a.number(12));
      p.softcap = static_cast<float>(a.number(13));
      p.sig_bias = static_cast<float>(a.number(15));
      p.out_scale = static_cast<float>(a.number(16));
      const Args m(&PyTuple_GET_ITEM(a.v[11], 0), PyTuple_GET_SIZE(a.v[11]), 5);
      p.win_left = m.integer(0);
      p.win_right = m.integer(1);
      p.block = m.integer(2);
      p.prefix = m.integer(3);
      p.dilation = m.integer(4);
      p.status = reinterpret_cast<int32_t *>(a.integer(20));
      p.workspace = ws.data_ptr();
      p.workspace_bytes = ws.numel();
      p.wait_limit_ns = static_cast<uint64_t>(a.integer(19));
      const int code = tree_pos != nullptr ? g_tree_attn(&p, tree_pos, tree_word, stream) : g_attn(&p, stream);
      if (code != CHIA_OK) return PyLong_FromLong(code);
      if (!a.none(17)) written(out);
    }
    PyObject *o = a.none(17) ? THPVariable_Wrap(out) : Py_NewRef(a.v[17]);
    if (!lse.defined()) return o;
    return Py_BuildValue("(NN)", o, THPVariable_Wrap(lse));
  });
}

// Addresses of libchia_attn.so's entry points, in the order below.
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject * {
    const Args a(args, nargs, 13);
    auto set = [&](auto &f, int i) {
      f = reinterpret_cast<std::decay_t<decltype(f)>>(static_cast<uintptr_t>(a.integer(i)));
    };
    set(g_tables, 0), set(g_release, 1), set(g_append, 2), set(g_attn, 3), set(g_bytes, 4), set(g_trim, 5);
    set(g_tree_tables, 6), set(g_tree_attn, 7), set(g_verify, 8), set(g_compact, 9);
    set(g_rope, 10), set(g_rope_bwd, 11), set(g_rope_bytes, 12);
    Py_RETURN_NONE;
  });
}

PyCFunction fast(PyObject *(*f)(PyObject *, PyObject *const *, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef kMethods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},
                          {"tables", fast(tables), METH_FASTCALL, nullptr},
                          {"append", fast(append), METH_FASTCALL, nullptr},
                          {"attention", fast(attention), METH_FASTCALL, nullptr},
                          {"tree_tables", fast(tree_tables), METH_FASTCALL, nullptr},
                          {"verify", fast(verify), METH_FASTCALL, nullptr},
                          {"compact", fast(compact), METH_FASTCALL, nullptr},
                          {"qk_norm_rope", fast(qk_norm_rope), METH_FASTCALL, nullptr},
                          {"qk_norm_rope_bwd", fast(qk_norm_rope_bwd), METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&kModule); }
