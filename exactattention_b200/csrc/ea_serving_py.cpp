// Python binding of the serving operators (include/exactattn_serving.h): checks the tensors, allocates the
// outputs on the current stream's pool, fills the argument structs and calls the C entries.
//
// A call through ctypes costs 20-25 us of interpreter time, several times what the small calls take on the
// GPU; this module's calls cost 3-6 us. serving.py holds the documented functions, which pass their
// arguments on by position. Wrong arguments raise ValueError, tensors off the GPU and CUDA errors RuntimeError.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/exactattn_serving.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void need(bool ok, const char* msg) {
  if (!ok) throw Refused(msg);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  // the operators record no graph: a gradient through them would be dropped without a word
  if (t.requires_grad() && c10::GradMode::is_enabled())
    throw Refused(std::string(name) + " requires grad, which the serving operators do not record (torch.no_grad, or detach it)");
  return t;
}

int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused(std::string(name) + " must be an integer");
  }
  return v;
}

constexpr int64_t ANY = -1;

// data of a contiguous tensor of the given type, device and shape (ANY: any extent), nullptr for None
template <typename... N>
void* flat(PyObject* o, const char* name, at::ScalarType type, const at::Device& dev, N... shape) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  const int64_t want[] = {(int64_t)shape...};
  bool ok = t.scalar_type() == type && t.device() == dev && t.is_contiguous() && t.dim() == (int64_t)sizeof...(N);
  for (size_t i = 0; ok && i < sizeof...(N); ++i) ok = want[i] == ANY || t.size((int64_t)i) == want[i];
  if (!ok) {
    std::string s = std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor on " + dev.str() + " of shape (";
    for (size_t i = 0; i < sizeof...(N); ++i) s += (i ? ", " : "") + (want[i] == ANY ? std::string("any") : std::to_string(want[i]));
    throw Refused(s + ")");
  }
  return t.data_ptr();
}
template <typename... N>
int32_t* ints(PyObject* o, const char* name, const at::Device& dev, N... shape) {
  return (int32_t*)flat(o, name, at::kInt, dev, shape...);
}
template <typename... N>
float* floats(PyObject* o, const char* name, const at::Device& dev, N... shape) {
  return (float*)flat(o, name, at::kFloat, dev, shape...);
}

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? EA_BF16 : t == at::kHalf ? EA_FP16 : t == at::kFloat ? EA_FP32 : -1;
}

// page table (batch, max_pages) int32 with contiguous rows
const at::Tensor& table(PyObject* o, const at::Device& dev, int64_t batch) {
  const at::Tensor& t = tensor(o, "page_table");
  need(t.scalar_type() == at::kInt && t.device() == dev && t.dim() == 2 && t.size(0) == batch &&
           (t.stride(1) == 1 || t.numel() <= batch),
       "page_table must be a (batch, max_pages) int32 tensor with contiguous rows on the other tensors' device");
  return t;
}

template <typename A>
void call(int (*fn)(const A*, void*), const A& a, const at::Device& dev) {
  const int rc = fn(&a, (void*)c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc == 0) return;
  const std::string msg = std::string(ea_serving_last_error()) + " (code " + std::to_string(rc) + ")";
  if (rc == -4) throw std::runtime_error(msg);
  throw Refused(msg);
}

void on_gpu(const at::Device& dev, const char* what) {
  if (!dev.is_cuda()) throw std::runtime_error(std::string(what) + " needs CUDA tensors (there is no CPU path)");
}

// An uninitialised tensor, without the dispatcher's share of at::empty.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

// `len` elements of a contiguous tensor from `off` on, sharing its storage.
at::Tensor part(const at::Tensor& t, int64_t off, int64_t len) {
  at::Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  v.unsafeGetTensorImpl()->set_storage_offset(t.storage_offset() + off);
  v.unsafeGetTensorImpl()->set_sizes_contiguous(len);
  return v;
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
  if (n != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  if (out)
    for (const at::Tensor& t : ts) {
      PyObject* w = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
      if (!w) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i++, w);
    }
  return out;
}

// context_lens, new_lens, page_table, free_pages, page_size, max_tokens, free_head, depths
PyObject* plan_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor& ctx = tensor(v[0], "context_lens");
    const at::Device dev = ctx.device();
    need(ctx.dim() == 1, "context_lens must be (batch,)");
    const int64_t batch = ctx.size(0), cap = integer(v[5], "max_tokens"), ps = integer(v[4], "page_size");
    need(cap >= 0 && cap < (1ll << 31) && ps > 0 && ps < (1ll << 31),
         "max_tokens must not be negative and page_size must be positive");
    ea_plan_step_t a = {};
    a.context_lens = ints(v[0], "context_lens", dev, ANY);
    a.new_lens = ints(v[1], "new_lens", dev, batch);
    const at::Tensor& tab = table(v[2], dev, batch);
    const at::Tensor& free_pages = tensor(v[3], "free_pages");
    a.page_table = (int32_t*)tab.data_ptr();
    a.free_pages = ints(v[3], "free_pages", dev, ANY);
    a.free_head = ints(v[6], "free_head", dev, 1);
    a.depths = ints(v[7], "depths", dev, cap);
    need(batch <= EA_PLAN_MAX_SEQS, "plan_step: more than EA_PLAN_MAX_SEQS sequences");
    on_gpu(dev, "plan_step");
    c10::cuda::OptionalCUDAGuard guard(dev);
    at::Tensor slots = fresh({cap}, at::kLong, dev);
    at::Tensor per_tok = fresh({2 * cap}, at::kInt, dev), per_seq = fresh({2 * batch + 3}, at::kInt, dev);
    a.slot_map = slots.data_ptr<int64_t>();
    a.positions = per_tok.data_ptr<int32_t>(), a.token_seq = a.positions + cap;
    a.q_start = per_seq.data_ptr<int32_t>(), a.seq_lens = a.q_start + batch + 1;
    a.next_free_head = a.seq_lens + batch, a.status = a.next_free_head + 1;
    a.table_stride = tab.stride(0);
    a.batch = (int)batch, a.max_pages = (int)tab.size(1), a.page_size = (int)ps;
    a.num_free = (int)free_pages.size(0), a.max_tokens = (int)cap;
    call(ea_plan_step_cuda, a, dev);
    return tuple_of({slots, part(per_tok, 0, cap), part(per_tok, cap, cap), part(per_seq, 0, batch + 1),
                     part(per_seq, batch + 1, batch), part(per_seq, 2 * batch + 1, 1), part(per_seq, 2 * batch + 2, 1)});
  });
}

// q, k, v, positions, inv_freq, axes, adjacent, inverse, slot_map, k_cache, v_cache
PyObject* rope(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded(nargs, 11, [&]() -> PyObject* {
    const bool hq = v[0] != Py_None, hk = v[1] != Py_None, append = v[8] != Py_None;
    need(hq || hk, "rope needs q or k");
    const at::Tensor& first = tensor(hq ? v[0] : v[1], "q");
    const at::Device dev = first.device();
    const at::ScalarType type = first.scalar_type();
    need(type_code(type) >= 0, "rope takes bfloat16, float16 or float32");
    need(first.dim() == 3, "q and k must be (tokens, heads, d)");
    const int64_t n = first.size(0), d = first.size(2);
    const auto heads = [&](PyObject* o, const char* name) -> const at::Tensor& {
      const at::Tensor& t = tensor(o, name);
      if (!(t.dim() == 3 && t.size(0) == n && t.size(2) == d && t.scalar_type() == type && t.device() == dev &&
            (t.stride(2) == 1 || d == 1)))
        throw Refused(std::string(name) + " must be a (tokens, heads, d) tensor like q, with contiguous channels");
      return t;
    };
    const at::Tensor& pos = tensor(v[3], "positions");
    const int64_t pd = pos.dim();
    need(pos.scalar_type() == at::kInt && pos.device() == dev && (pd == 1 || pd == 2) && pos.size(pd - 1) == n &&
             (n <= 1 || pos.stride(pd - 1) == 1),
         "positions must be int32, (tokens,) or (axes, tokens), on q's device");
    const at::Tensor& freq = tensor(v[4], "inv_freq");
    need(freq.dim() == 1 && 2 * freq.size(0) <= d, "inv_freq must be (rot / 2,) with rot at most d");
    const int64_t half = freq.size(0);
    ea_rope_t a = {};
    a.inv_freq = floats(v[4], "inv_freq", dev, half);
    a.axes = ints(v[5], "axes", dev, half);
    a.positions = pos.data_ptr<int32_t>();
    a.axis_stride = pd == 2 ? pos.stride(0) : 0, a.num_axes = pd == 2 ? (int)pos.size(0) : 1;
    a.tokens = n, a.d = (int)d, a.rot = (int)(2 * half), a.dtype = type_code(type);
    a.adjacent = v[6] == Py_True, a.inverse = v[7] == Py_True;
    if (hq) {
      const at::Tensor& q = heads(v[0], "q");
      a.q = q.data_ptr(), a.q_stride = q.stride(0), a.q_head_stride = q.stride(1), a.q_heads = (int)q.size(1);
    }
    if (hk) {
      const at::Tensor& k = heads(v[1], "k");
      a.k = k.data_ptr(), a.k_stride = k.stride(0), a.k_head_stride = k.stride(1), a.kv_heads = (int)k.size(1);
    }
    if (append) {
      need(hk && v[2] != Py_None, "rope_append needs k and v");
      const at::Tensor& w = heads(v[2], "v");
      need(w.size(1) == a.kv_heads, "rope_append needs k and v of one shape");
      a.v = w.data_ptr(), a.v_stride = w.stride(0), a.v_head_stride = w.stride(1);
      a.slot_map = (const int64_t*)flat(v[8], "slot_map", at::kLong, dev, n);
      const at::Tensor &kc = tensor(v[9], "k_cache"), &vc = tensor(v[10], "v_cache");
      for (const at::Tensor* c : {&kc, &vc})
        need(c->dim() == 4 && c->sizes() == kc.sizes() && c->size(1) == a.kv_heads && c->size(3) == d &&
                 c->scalar_type() == type && c->device() == dev && (c->stride(3) == 1 || d == 1),
             "the caches must be (pages, kv_heads, page_size, d) tensors of q's type with contiguous channels");
      a.k_cache = kc.data_ptr(), a.v_cache = vc.data_ptr();
      a.k_page_stride = kc.stride(0), a.k_cache_head_stride = kc.stride(1), a.k_row_stride = kc.stride(2);
      a.v_page_stride = vc.stride(0), a.v_cache_head_stride = vc.stride(1), a.v_row_stride = vc.stride(2);
      a.page_size = (int)kc.size(2), a.num_slots = kc.size(0) * kc.size(2);
    }
    on_gpu(dev, "rope");
    c10::cuda::OptionalCUDAGuard guard(dev);
    at::Tensor q_out, k_out;
    if (hq) q_out = fresh({n, a.q_heads, d}, type, dev), a.q_out = q_out.data_ptr();
    if (hk && !append) k_out = fresh({n, a.kv_heads, d}, type, dev), a.k_out = k_out.data_ptr();
    call(ea_rope_cuda, a, dev);
    return tuple_of({q_out, k_out});
  });
}

// q, k_cache, v_cache, page_table, seq_lens, q_start, alpha, tree_mask, max_new, want_lse, out
PyObject* tree_attention(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded(nargs, 11, [&]() -> PyObject* {
    const at::Tensor &q = tensor(v[0], "q"), &kc = tensor(v[1], "k_cache"), &vc = tensor(v[2], "v_cache");
    const at::Device dev = q.device();
    const at::ScalarType type = q.scalar_type();
    need(type == at::kBFloat16 || type == at::kHalf, "tree_attention takes bfloat16 or float16");
    need(q.dim() == 3 && (q.stride(2) == 1 || q.size(2) == 1), "q must be (tokens, q_heads, d) with contiguous channels");
    const int64_t n = q.size(0), hq = q.size(1), d = q.size(2);
    for (const at::Tensor* c : {&kc, &vc})
      need(c->dim() == 4 && c->sizes() == kc.sizes() && c->size(3) == d && c->scalar_type() == type && c->device() == dev &&
               (c->stride(3) == 1 || d == 1),
           "the caches must be (pages, kv_heads, page_size, d) tensors of q's type with contiguous channels");
    const at::Tensor& lens = tensor(v[4], "seq_lens");
    need(lens.dim() == 1, "seq_lens must be (batch,)");
    const int64_t batch = lens.size(0);
    const at::Tensor& tab = table(v[3], dev, batch);
    ea_tree_attention_t a = {};
    a.seq_lens = ints(v[4], "seq_lens", dev, ANY);
    a.q_start = ints(v[5], "q_start", dev, batch + 1);
    a.alpha = (float)PyFloat_AsDouble(v[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      throw Refused("alpha must be a number");
    }
    if (v[7] != Py_None) {
      a.tree_mask = ints(v[7], "tree_mask", dev, n, ANY);
      a.mask_words = (int)THPVariable_Unpack(v[7]).size(1);
    }
    at::Tensor out, lse, ws;
    if (v[10] != Py_None) {
      out = tensor(v[10], "out");
      need(out.sizes() == q.sizes() && out.scalar_type() == type && out.device() == dev && out.is_contiguous(),
           "out must be a contiguous tensor like q");
    }
    on_gpu(dev, "tree_attention");
    c10::cuda::OptionalCUDAGuard guard(dev);
    if (!out.defined()) out = fresh({n, hq, d}, type, dev);
    if (v[9] == Py_True) lse = fresh({n, hq}, at::kFloat, dev), a.lse = lse.data_ptr<float>();
    a.q = q.data_ptr(), a.q_stride = q.stride(0), a.q_head_stride = q.stride(1);
    a.k_cache = kc.data_ptr(), a.k_page_stride = kc.stride(0), a.k_head_stride = kc.stride(1), a.k_row_stride = kc.stride(2);
    a.v_cache = vc.data_ptr(), a.v_page_stride = vc.stride(0), a.v_head_stride = vc.stride(1), a.v_row_stride = vc.stride(2);
    a.page_table = (const int32_t*)tab.data_ptr(), a.table_stride = tab.stride(0);
    a.out = out.data_ptr();
    a.tokens = n, a.num_pages = kc.size(0);
    a.batch = (int)batch, a.q_heads = (int)hq, a.kv_heads = (int)kc.size(1), a.d = (int)d;
    a.page_size = (int)kc.size(2), a.max_pages = (int)tab.size(1), a.dtype = type_code(type);
    a.max_new = v[8] == Py_None ? (int)n : (int)integer(v[8], "max_new");
    if (n && batch) {
      const int64_t bytes = ea_tree_attention_workspace(&a);
      if (bytes < 0) throw Refused(ea_serving_last_error());
      ws = fresh({bytes}, at::kByte, dev);
      a.workspace = ws.data_ptr();
    }
    call(ea_tree_attention_cuda, a, dev);
    return tuple_of({out, lse});
  });
}

// logits, row_seq, history, history_lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values,
// allowed_bits, mask_rows, draft_tokens, q_start, tree_mask, out
PyObject* process_logits(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded(nargs, 16, [&]() -> PyObject* {
    const at::Tensor& x = tensor(v[0], "logits");
    const at::Device dev = x.device();
    need(type_code(x.scalar_type()) >= 0, "process_logits takes bfloat16, float16 or float32");
    need(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1), "logits must be (rows, vocab) with contiguous rows");
    const int64_t rows = x.size(0), vocab = x.size(1);
    need(vocab < (1ll << 31), "process_logits: vocabulary above its limit");
    at::Tensor out;
    if (v[15] != Py_None) {
      out = tensor(v[15], "out");
      need(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.device() == dev &&
               (out.stride(1) == 1 || vocab <= 1),
           "out must be a tensor like logits with contiguous rows");
    }
    int64_t batch = -1;
    for (int i : {2, 5, 6, 7, 8})
      if (v[i] != Py_None) {
        const at::Tensor& t = tensor(v[i], "a sequences' tensor");
        need(t.dim() >= 1 && (batch < 0 || t.size(0) == batch), "the sequences' tensors differ in length");
        batch = t.size(0);
      }
    // Where nothing says how many sequences there are, masks alone are left to apply: any row_seq may be one.
    if (batch < 0) batch = v[13] != Py_None ? tensor(v[13], "q_start").numel() - 1 : v[1] == Py_None ? rows : EA_LOGITS_MAX_SEQS;
    need(v[1] != Py_None || batch == rows, "without row_seq there must be one row a sequence");
    need(batch >= 0 && batch <= EA_LOGITS_MAX_SEQS, "process_logits: more sequences than its limit");
    ea_process_logits_t a = {};
    a.row_seq = ints(v[1], "row_seq", dev, rows);
    if (v[2] != Py_None) {
      need(v[3] != Py_None, "history needs history_lens");
      a.history = ints(v[2], "history", dev, batch, ANY);
      const int64_t w = THPVariable_Unpack(v[2]).size(1);
      need(w <= EA_LOGITS_MAX_HISTORY, "process_logits: history above its limit");
      a.history_stride = w, a.max_history = (int)w;
      a.history_lens = ints(v[3], "history_lens", dev, batch);
      a.prompt_lens = ints(v[4], "prompt_lens", dev, batch);
    }
    a.repetition = floats(v[5], "repetition", dev, batch);
    a.frequency = floats(v[6], "frequency", dev, batch);
    a.presence = floats(v[7], "presence", dev, batch);
    if (v[8] != Py_None) {
      need(v[9] != Py_None, "bias_ids needs bias_values");
      a.bias_ids = ints(v[8], "bias_ids", dev, batch, ANY);
      const int64_t w = THPVariable_Unpack(v[8]).size(1);
      need(w <= EA_LOGITS_MAX_BIASES, "process_logits: biases above their limit");
      a.num_biases = (int)w;
      a.bias_values = floats(v[9], "bias_values", dev, batch, w);
    }
    if (v[10] != Py_None) {
      a.allowed_bits = ints(v[10], "allowed_bits", dev, ANY, ANY);
      const at::Tensor& t = THPVariable_Unpack(v[10]);
      need(t.size(1) >= (vocab + 31) / 32, "allowed_bits needs a bit for every token");
      need(v[11] != Py_None || t.size(0) >= rows, "without mask_rows there must be one mask a row");
      a.num_masks = (int)t.size(0), a.mask_stride = t.size(1);
      a.mask_rows = ints(v[11], "mask_rows", dev, rows);
    }
    if (v[12] != Py_None) {
      need(v[13] != Py_None, "draft_tokens needs q_start");
      a.draft_tokens = ints(v[12], "draft_tokens", dev, rows);
      a.q_start = ints(v[13], "q_start", dev, batch + 1);
      if (v[14] != Py_None) {
        a.tree_mask = ints(v[14], "tree_mask", dev, rows, ANY);
        a.tree_words = (int)THPVariable_Unpack(v[14]).size(1);
      }
    }
    on_gpu(dev, "process_logits");
    c10::cuda::OptionalCUDAGuard guard(dev);
    if (!out.defined()) out = fresh({rows, vocab}, x.scalar_type(), dev);
    a.logits = x.data_ptr(), a.logits_stride = x.stride(0), a.out = out.data_ptr(), a.out_stride = out.stride(0);
    a.rows = rows, a.vocab = (int)vocab, a.batch = (int)batch, a.dtype = type_code(x.scalar_type());
    call(ea_process_logits_cuda, a, dev);
    return v[15] != Py_None ? Py_NewRef(v[15]) : THPVariable_Wrap(out);
  });
}

PyMethodDef methods[] = {{"plan_step", (PyCFunction)(void (*)())plan_step, METH_FASTCALL, nullptr},
                         {"rope", (PyCFunction)(void (*)())rope, METH_FASTCALL, nullptr},
                         {"tree_attention", (PyCFunction)(void (*)())tree_attention, METH_FASTCALL, nullptr},
                         {"process_logits", (PyCFunction)(void (*)())process_logits, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__serving_native() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", "built against torch " EA_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
