// pybind11 module `llcompiler_`: the reference's Python-facing native module
// (src/Pybind/Entrance.cpp:69-120) re-bound onto the C ABI of llc_runtime.h.  Same submodules
// (tensor, compiler, executor), same class and method names, same argument order.  A non-zero
// status from the C ABI becomes a Python RuntimeError (the reference logs and carries on,
// include/llcompiler/Support/Logger.h:126-134).
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cmath>
#include <cstring>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <vector>

#include "llc_cuda.h"
#include "llc_runtime.h"

namespace py = pybind11;

namespace {

void check(int rc) { if (rc != LLC_OK) throw std::runtime_error(std::string("[llc status ") + std::to_string(rc) + "] " + llc_last_error()); }

// llc::compiler::Tensor (include/llcompiler/Compiler/Tensor.h:35-48) plus a device ordinal.
struct Tensor {
  uintptr_t data = 0, base = 0;
  int type = LLC_FLOAT32;
  int64_t offset = 0;
  std::vector<int64_t> size, stride;
  int device = -1;
  Tensor() {}
  Tensor(uintptr_t data_ptr, uintptr_t base_ptr, int type_, int64_t offset_, std::vector<int64_t> size_, std::vector<int64_t> stride_, int device_ = -1)
      : data(data_ptr), base(base_ptr), type(type_), offset(offset_), size(std::move(size_)), stride(std::move(stride_)), device(device_) {}
  LlcTensor desc() const { return LlcTensor{reinterpret_cast<void*>(data), type, device, (int32_t)size.size(), size.data(), stride.data()}; }
  void print() const {
    std::string s = "Tensor(data=" + std::to_string(data) + ", type=" + std::to_string(type) + ", device=" + std::to_string(device) + ", size=[";
    for (size_t i = 0; i < size.size(); ++i) s += (i ? "," : "") + std::to_string(size[i]);
    py::print(s + "])");
  }
};

// Element size and struct-module format of a dtype code (the reference's get_itemsize / get_format,
// src/Pybind/Entrance.cpp:27-58, plus the two 16-bit floats).
py::ssize_t itemSize(int type) {
  switch (type) {
    case LLC_INT8: case LLC_INT1: return 1;
    case LLC_INT16: case LLC_FLOAT16: case LLC_BFLOAT16: return 2;
    case LLC_INT32: case LLC_FLOAT32: return 4;
    default: return 8;
  }
}
std::string formatOf(int type) {
  switch (type) {
    case LLC_INT8: return "b"; case LLC_INT1: return "?"; case LLC_INT16: return "h"; case LLC_INT32: return "i"; case LLC_INT64: return "q";
    case LLC_FLOAT32: return "f"; case LLC_FLOAT64: return "d"; case LLC_FLOAT16: return "e";
    case LLC_BFLOAT16: return "H";      // no struct code for bf16: exposed as its 16-bit pattern
  }
  throw std::runtime_error("Tensor: unknown element type code " + std::to_string(type));
}
// Buffer view of a HOST tensor (the reference's tensors are always host memory, src/Pybind/Entrance.cpp:80-91);
// device memory cannot be read through the buffer protocol.
py::buffer_info bufferOf(Tensor& t) {
  if (t.device >= 0) throw std::runtime_error("Tensor: device memory has no buffer view; copy the torch tensor to the host first");
  std::vector<py::ssize_t> shape(t.size.begin(), t.size.end()), strides;
  for (auto s : t.stride) strides.push_back((py::ssize_t)s * itemSize(t.type));
  return py::buffer_info(reinterpret_cast<void*>(t.data), itemSize(t.type), formatOf(t.type), (py::ssize_t)shape.size(), shape, strides);
}

// The reference's executor.get_tool (src/Compiler/Command.cpp:13-15 over ToolPath.h.in:19-24) names the external
// programs its pipeline shells out to.  This backend runs no subprocess: "llc-opt" is the text-IR driver module, "cxx"
// the host compiler the build used; the LLVM tools have no counterpart and raise, as an unknown name does there.
std::string getTool(const std::string& name) {
  if (name == "llc-opt") return "python -m llcompiler_b200.llc_opt";
  if (name == "cxx") return "g++";
  throw py::index_error("no tool '" + name + "': the CUDA pipeline runs in-process and has no LLVM tool chain (opt, llc, llc-translate)");
}

// llc::compiler::CompileOptions (include/llcompiler/Compiler/CompileOption.h:39-71)
struct CompileOptions {
  std::string mode = "inference", target = "sm_100a", pipeline = "cuda", global_layout = "NCHW", log_root, log_level = "debug", cpu, mtriple, precision = "auto";
  bool mlir_passes = false, llvm_passes = false;
  LlcOptions c() const { return LlcOptions{mode.c_str(), target.c_str(), pipeline.c_str(), global_layout.c_str(), log_root.c_str(), log_level.c_str(), cpu.c_str(), mtriple.c_str(), precision.c_str()}; }
};

struct Compiler {
  std::string compile_mlir_to_shared_lib(const std::string& text, const CompileOptions& o) {
    char path[1024];
    LlcOptions c = o.c();
    check(llc_compile(text.c_str(), &c, path, sizeof path));
    return path;
  }
  std::string run_pass(const std::string& text, const std::string& pass, const CompileOptions& o) {
    const char* out = nullptr;
    LlcOptions c = o.c();
    check(llc_run_pass(text.c_str(), pass.c_str(), &c, &out));
    return out;
  }
};

// llc::compiler::Execution (src/Compiler/Execution.cpp:10-66)
struct Execution {
  LlcExec* exec = nullptr;
  ~Execution() { if (exec) llc_free(exec); }
  void load(const std::string& path, int device, const std::string& weight_dir) {
    if (exec) throw std::runtime_error("Execution.load may be called once per object");
    check(llc_load_from(path.c_str(), weight_dir.empty() ? nullptr : weight_dir.c_str(), device, &exec));
  }
  bool loaded_from_pool() const { need(); return llc_loaded_from_pool(exec) == 1; }
  void need() const { if (!exec) throw std::runtime_error("Execution.load has not been called"); }
  void run_impl(const std::vector<int64_t>& symbols, std::vector<Tensor*>& in, std::vector<Tensor*>& out, uintptr_t stream) {
    need();
    std::vector<LlcTensor> ci, co;
    for (auto* t : in) ci.push_back(t->desc());
    for (auto* t : out) co.push_back(t->desc());
    int rc;
    {
      py::gil_scoped_release release;
      rc = llc_run(exec, symbols.data(), (int)symbols.size(), ci.data(), (int)ci.size(), co.data(), (int)co.size(), reinterpret_cast<void*>(stream));
    }
    check(rc);
  }
  void run(std::vector<Tensor*> in, std::vector<Tensor*> out, uintptr_t stream) { run_impl({}, in, out, stream); }
  void run_with_symbols(std::vector<int64_t> symbols, std::vector<Tensor*> in, std::vector<Tensor*> out, uintptr_t stream) { run_impl(symbols, in, out, stream); }
  std::vector<std::pair<std::vector<int64_t>, int>> output_shapes(std::vector<int64_t> symbols, std::vector<Tensor*> in) {
    need();
    std::vector<LlcTensor> ci;
    for (auto* t : in) ci.push_back(t->desc());
    std::vector<std::pair<std::vector<int64_t>, int>> res;
    for (int k = 0; k < llc_num_outputs(exec); ++k) {
      int64_t sizes[8]; int32_t rank = 0, dtype = 0;
      check(llc_output_shape(exec, symbols.data(), (int)symbols.size(), ci.data(), (int)ci.size(), k, sizes, &rank, &dtype));
      res.emplace_back(std::vector<int64_t>(sizes, sizes + rank), dtype);
    }
    return res;
  }
  std::string profile(std::vector<int64_t> symbols, std::vector<Tensor*> in, std::vector<Tensor*> out, int reps, uintptr_t stream) {
    need();
    std::vector<LlcTensor> ci, co;
    for (auto* t : in) ci.push_back(t->desc());
    for (auto* t : out) co.push_back(t->desc());
    std::string report(1 << 20, '\0');
    check(llc_profile(exec, symbols.data(), (int)symbols.size(), ci.data(), (int)ci.size(), co.data(), (int)co.size(), reps,
                      reinterpret_cast<void*>(stream), &report[0], report.size()));
    report.resize(strlen(report.c_str()));
    return report;
  }
  // Raises when a kernel of an earlier call recorded a failure (see llc_status); returns the three words otherwise.
  std::vector<int> status() {
    need();
    int32_t w[3] = {0, 0, 0};
    int rc;
    {
      py::gil_scoped_release release;
      rc = llc_status(exec, w);
    }
    check(rc);
    return {w[0], w[1], w[2]};
  }
  int num_inputs() const { need(); return llc_num_inputs(exec); }
  int num_outputs() const { need(); return llc_num_outputs(exec); }
  int num_symbols() const { need(); return llc_num_symbols(exec); }
  int64_t last_launch_count() const { need(); return llc_last_launch_count(exec); }
  int64_t arena_bytes() const { need(); return llc_arena_bytes(exec); }
};

// ---- Operators of the kernel library that a serving loop calls on device tensors directly, without a compiled plan
// (llcompiler_b200/executor/paged.py).  A decoding step makes a handful of such calls of a few microseconds each, so the checks are
// made here: what a tensor says of itself is read through the interpreter once, nothing links against the tensor library.
py::object got(PyObject* o) { if (!o) throw py::error_already_set(); return py::reinterpret_steal<py::object>(o); }

struct Torch {
  py::object tensor, emptyLike, empty, stream, gradEnabled, forwardAd, wrote;
  py::object f32, f16, bf16, f64, i32, i64;
  PyObject* nShape, *nStride, *nDtype, *nPtr, *nDevice, *nGrad, *nDeviceOf, *nLevel, *kwEmpty;
  Torch() {
    py::module_ t = py::module_::import("torch"), c = py::module_::import("torch._C");
    tensor = t.attr("Tensor"); emptyLike = t.attr("empty_like"); empty = t.attr("empty"); gradEnabled = t.attr("is_grad_enabled");
    stream = c.attr("_cuda_getCurrentRawStream"); forwardAd = py::module_::import("torch.autograd.forward_ad");
    wrote = c.attr("_increment_version");
    f32 = t.attr("float32"); f16 = t.attr("float16"); bf16 = t.attr("bfloat16"); f64 = t.attr("float64"); i32 = t.attr("int32"); i64 = t.attr("int64");
    nShape = PyUnicode_InternFromString("shape"); nStride = PyUnicode_InternFromString("stride"); nDtype = PyUnicode_InternFromString("dtype");
    nPtr = PyUnicode_InternFromString("data_ptr"); nDevice = PyUnicode_InternFromString("get_device"); nGrad = PyUnicode_InternFromString("requires_grad");
    nDeviceOf = PyUnicode_InternFromString("device"); nLevel = PyUnicode_InternFromString("_current_level");
    kwEmpty = PyTuple_Pack(2, nDtype, nDeviceOf);
  }
  // Whether a dual level is open (-1: none is): asked once a call, the level is the process's.
  mutable bool dualLevel = false;
  void look() const { dualLevel = PyLong_AsLong(got(PyObject_GetAttr(forwardAd.ptr(), nLevel)).ptr()) >= 0; }
  int code(PyObject* d) const {
    if (d == bf16.ptr()) return LLC_BFLOAT16;
    if (d == f16.ptr()) return LLC_FLOAT16;
    if (d == f32.ptr()) return LLC_FLOAT32;
    if (d == i32.ptr()) return LLC_INT32;
    if (d == i64.ptr()) return LLC_INT64;
    if (d == f64.ptr()) return LLC_FLOAT64;
    return -1;
  }
};
// Guarded by the interpreter's lock alone: making one runs Python code, which may hand the lock to another thread, and a thread that waited there for
// a C++ guard would keep it.  Two first calls at once make two, of which one is kept.  Never destroyed: the interpreter may be gone by then.
const Torch& torch() {
  static Torch* t = nullptr;
  if (!t) {
    Torch* made = new Torch();
    if (!t) t = made;
  }
  return *t;
}

int64_t number(const char* name, PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) { PyErr_Clear(); throw py::type_error(std::string(name) + ": expected a whole number of 64 bits"); }
  return x;
}

// One operand.  `name` goes into the message when something does not fit.
struct Operand {
  const char* name;
  int rank = 0, dtype = -1, device = -1;
  int64_t n[4] = {1, 1, 1, 1}, s[4] = {0, 0, 0, 0};
  uintptr_t ptr = 0;
  [[noreturn]] void bad(const std::string& what) const { throw py::value_error(std::string(name) + ": " + what); }
  std::string shape() const {
    std::string r = "(";
    for (int i = 0; i < rank; ++i) r += (i ? ", " : "") + std::to_string(n[i]);
    return r + ")";
  }
  // The caller's tensor, checked.  Whole numbers never require a gradient: `index` skips that question.
  Operand(const char* name_, py::handle h, int least, int most, bool index = false) : name(name_) {
    const Torch& t = torch();
    PyObject* o = h.ptr();
    if (!PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(t.tensor.ptr()))) throw py::type_error(std::string(name) + ": expected a tensor, got " + Py_TYPE(o)->tp_name);
    py::object sh = got(PyObject_GetAttr(o, t.nShape)), st = got(PyObject_CallMethodNoArgs(o, t.nStride)), dt = got(PyObject_GetAttr(o, t.nDtype)),
               dv = got(PyObject_CallMethodNoArgs(o, t.nDevice)), pt = got(PyObject_CallMethodNoArgs(o, t.nPtr));
    rank = (int)PyTuple_GET_SIZE(sh.ptr());
    if (rank < least || rank > most) throw py::value_error(std::string(name) + ": expected " + std::to_string(least) + " dims, got " + std::to_string(rank));
    for (int i = 0; i < rank; ++i) { n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(sh.ptr(), i)); s[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(st.ptr(), i)); }
    dtype = t.code(dt.ptr());
    device = (int)PyLong_AsLong(dv.ptr());
    ptr = (uintptr_t)PyLong_AsUnsignedLongLong(pt.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    if (device < 0) bad("expected a CUDA tensor; there is no CPU fallback");
    if (index) return;
    if (got(PyObject_GetAttr(o, t.nGrad)).ptr() == Py_True && t.gradEnabled().cast<bool>()) bad("inference only, it requires a gradient");
    // a dual tensor does not say so itself
    if (t.dualLevel && !t.forwardAd.attr("unpack_dual")(h).attr("tangent").is_none()) bad("inference only, it carries a forward-mode tangent");
  }
  // A tensor just made like `l`: only its strides and its address are news.
  Operand(const char* name_, py::handle h, const Operand& l) : name(name_) {
    const Torch& t = torch();
    py::object st = got(PyObject_CallMethodNoArgs(h.ptr(), t.nStride)), pt = got(PyObject_CallMethodNoArgs(h.ptr(), t.nPtr));
    rank = l.rank; dtype = l.dtype; device = l.device;
    for (int i = 0; i < rank; ++i) { n[i] = l.n[i]; s[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(st.ptr(), i)); }
    ptr = (uintptr_t)PyLong_AsUnsignedLongLong(pt.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
  }
  void on(int dev) const { if (device != dev) bad("on cuda:" + std::to_string(device) + ", expected cuda:" + std::to_string(dev)); }
  void type(int want, const char* said) const { if (dtype != want) bad(std::string("expected ") + said); }
  void written() const { for (int i = 0; i < rank; ++i) if (n[i] > 1 && s[i] == 0) bad("an output may not repeat its elements (stride 0)"); }
  void unit(int dim, const char* what) const { if (n[dim] > 1 && s[dim] != 1) bad(std::string(what) + " must have unit stride"); }
};
// [tokens, heads, head_dim]
Operand rows(const char* name, py::handle h) { Operand o(name, h, 3, 3); o.unit(2, "the head dim"); return o; }
Operand rowsLike(const char* name, py::handle h, const Operand& first) {
  Operand o = rows(name, h);
  o.on(first.device);
  if (o.dtype != first.dtype) o.bad(std::string("expected the type of ") + first.name);
  return o;
}
Operand firstRows(const char* name, py::handle h) {
  Operand o = rows(name, h);
  if (o.dtype != LLC_FLOAT32 && o.dtype != LLC_BFLOAT16 && o.dtype != LLC_FLOAT16) o.bad("expected float32, bfloat16 or float16");
  return o;
}
// The result's tensor: the caller's, or a new one.
Operand output(const char* name, py::object& out, py::handle like, const Operand& l) {
  if (out.is_none()) {
    out = got(PyObject_CallOneArg(torch().emptyLike.ptr(), like.ptr()));
    Operand o(name, out, l);
    if (l.n[2] <= 1 || o.s[2] == 1) return o;
    out = torch().empty(like.attr("shape"), py::arg("dtype") = like.attr("dtype"), py::arg("device") = like.attr("device"));
  }
  Operand o = rowsLike(name, out, l);
  for (int i = 0; i < 3; ++i) if (o.n[i] != l.n[i]) o.bad("expected shape " + l.shape() + ", got " + o.shape());
  o.written();
  return o;
}

struct Turns { uintptr_t positions = 0, freq = 0; int posType = LLC_INT64, axes = 0; int64_t posStride = 0, pairs = 0; int32_t sections[LLC_ROTARY_MAX_AXES] = {0, 0, 0, 0}; };
Turns turns(py::handle positions, py::handle freq, py::handle sections, int64_t tokens, int64_t d, int device) {
  Turns t;
  Operand f("inv_freq", freq, 1, 1);
  f.on(device);
  f.type(LLC_FLOAT64, "float64");
  f.unit(0, "it");
  t.freq = f.ptr;
  t.pairs = f.n[0];
  if (t.pairs < 1 || 2 * t.pairs > d) f.bad(std::to_string(t.pairs) + " pairs do not fit a head of " + std::to_string(d));
  if (sections.is_none()) {
    t.axes = 1;
    t.sections[0] = (int32_t)t.pairs;
  } else {
    py::object list = got(PySequence_Fast(sections.ptr(), "sections: expected a sequence of numbers"));
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.ptr());
    int64_t sum = 0;
    bool fits = n >= 1 && n <= LLC_ROTARY_MAX_AXES;
    for (Py_ssize_t i = 0; fits && i < n; ++i) {
      const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(list.ptr(), i));
      if (x == -1 && PyErr_Occurred()) throw py::error_already_set();
      fits = x >= 0 && x <= t.pairs;
      if (fits) { t.sections[i] = (int32_t)x; sum += x; }
    }
    if (!fits || sum != t.pairs) throw py::value_error("sections: expected 1 to 4 numbers that add up to " + std::to_string(t.pairs) + " pairs");
    t.axes = (int)n;
  }
  if (positions.is_none()) return t;
  Operand p("positions", positions, 1, 2, true);
  p.on(device);
  if (p.dtype != LLC_INT32 && p.dtype != LLC_INT64) p.bad("expected int32 or int64");
  const int last = p.rank - 1;
  if (p.n[last] != tokens || (last ? p.n[0] : 1) != t.axes) p.bad("expected shape (" + std::to_string(t.axes) + ", " + std::to_string(tokens) + "), got " + p.shape());
  p.unit(last, "the tokens");
  t.positions = p.ptr; t.posType = p.dtype; t.posStride = last ? p.s[0] : 0;
  return t;
}

struct Batch { int64_t size, width, stride; const int32_t *table, *start, *len; int32_t* bad; };
Batch batchOf(py::handle table, py::handle start, py::handle len, py::handle bad, int device) {
  Operand t("page_table", table, 2, 2, true), s("q_start", start, 1, 1, true), l("kv_len", len, 1, 1, true);
  for (const Operand* o : {&t, &s, &l}) { o->on(device); o->type(LLC_INT32, "int32"); o->unit(o->rank - 1, "the last dim"); }
  if (s.n[0] != t.n[0] + 1) s.bad("expected " + std::to_string(t.n[0] + 1) + " entries, got " + std::to_string(s.n[0]));
  if (l.n[0] != t.n[0]) l.bad("expected " + std::to_string(t.n[0]) + " entries, got " + std::to_string(l.n[0]));
  Batch b{t.n[0], t.n[1], t.s[0], reinterpret_cast<const int32_t*>(t.ptr), reinterpret_cast<const int32_t*>(s.ptr), reinterpret_cast<const int32_t*>(l.ptr), nullptr};
  if (!bad.is_none()) {
    Operand x("bad_pages", bad, 1, 1, true);
    x.on(device);
    x.type(LLC_INT32, "int32");
    if (x.n[0] != 1) x.bad("expected one counter");
    b.bad = reinterpret_cast<int32_t*>(x.ptr);
  }
  return b;
}
Operand cacheOf(const char* name, py::handle h, const Operand& first) {
  Operand c(name, h, 4, 4);
  c.on(first.device);
  if (c.dtype != first.dtype) c.bad(std::string("expected the type of ") + first.name);
  c.unit(3, "the head dim");
  if (c.n[1] < 1 || c.n[2] < 1) c.bad("empty pages, shape " + c.shape());
  return c;
}
void sameShape(const Operand& a, const Operand& b) {
  for (int i = 0; i < a.rank; ++i) if (a.n[i] != b.n[i]) b.bad("expected shape " + a.shape() + ", got " + b.shape());
}
void* streamOf(int device) {
  py::object d = got(PyLong_FromLong(device)), s = got(PyObject_CallOneArg(torch().stream.ptr(), d.ptr()));
  return PyLong_AsVoidPtr(s.ptr());
}
// Tells autograd of the caller's tensors that a call has written: a graph that has saved one of them raises then instead of using new values.
void wrote(std::initializer_list<PyObject*> tensors) {
  py::tuple t(tensors.size());
  Py_ssize_t i = 0;
  for (PyObject* x : tensors) { Py_INCREF(x); PyTuple_SET_ITEM(t.ptr(), i++, x); }
  got(PyObject_CallOneArg(torch().wrote.ptr(), t.ptr()));
}
template <typename T = void> T* at(uintptr_t p) { return reinterpret_cast<T*>(p); }

py::object rotary(py::handle x, py::handle positions, py::handle freq, py::handle sections, bool interleaved, py::object out) {
  Operand a = firstRows("x", x);
  if (positions.is_none()) throw py::value_error("positions: required");
  const Turns t = turns(positions, freq, sections, a.n[0], a.n[2], a.device);
  const bool given = !out.is_none();
  const Operand o = output("out", out, x, a);
  LlcRotaryParams p{};
  p.x = at(a.ptr); p.out = at(o.ptr); p.positions = at(t.positions); p.inv_freq = at<const double>(t.freq);
  p.dtype = a.dtype; p.pos_dtype = t.posType; p.tokens = a.n[0]; p.heads = a.n[1]; p.d = a.n[2]; p.pairs = t.pairs;
  p.x_st = a.s[0]; p.x_sh = a.s[1]; p.o_st = o.s[0]; p.o_sh = o.s[1]; p.pos_sa = t.posStride; p.axes = t.axes; p.interleaved = interleaved;
  std::memcpy(p.sections, t.sections, sizeof p.sections);
  check(llc_cuda_rotary(&p, streamOf(a.device)));
  if (given) wrote({out.ptr()});
  return out;
}

py::object kvAppend(py::handle k, py::handle v, py::handle kCache, py::handle vCache, py::handle table, py::handle start, py::handle len, py::handle q, py::handle positions,
                    py::handle freq, py::handle sections, bool interleaved, py::object qOut, py::handle bad) {
  Operand a = firstRows("k", k), b = rowsLike("v", v, a), kc = cacheOf("k_cache", kCache, a), vc = cacheOf("v_cache", vCache, a);
  sameShape(a, b);
  sameShape(kc, vc);
  kc.written();
  vc.written();
  if (a.n[1] != kc.n[2] || a.n[2] != kc.n[3]) a.bad("expected [tokens, " + std::to_string(kc.n[2]) + ", " + std::to_string(kc.n[3]) + "], got " + a.shape());
  const Batch s = batchOf(table, start, len, bad, a.device);
  LlcKvAppendParams p{};
  const bool given = !qOut.is_none();
  if (!q.is_none()) {
    Operand x = rowsLike("q", q, a);
    if (x.n[0] != a.n[0] || x.n[2] != a.n[2]) x.bad("expected [" + std::to_string(a.n[0]) + ", heads, " + std::to_string(a.n[2]) + "], got " + x.shape());
    const Operand o = output("q_out", qOut, q, x);
    p.q = at(x.ptr); p.q_out = at(o.ptr); p.heads = x.n[1]; p.q_st = x.s[0]; p.q_sh = x.s[1]; p.qo_st = o.s[0]; p.qo_sh = o.s[1];
  } else if (given) {
    throw py::value_error("q_out: no queries were given");
  }
  if (!freq.is_none()) {
    const Turns t = turns(positions, freq, sections, a.n[0], a.n[2], a.device);
    p.positions = at(t.positions); p.inv_freq = at<const double>(t.freq); p.pos_dtype = t.posType; p.pairs = t.pairs; p.pos_sa = t.posStride; p.axes = t.axes;
    std::memcpy(p.sections, t.sections, sizeof p.sections);
  } else if (!positions.is_none() || !sections.is_none()) {
    throw py::value_error("positions and sections: no inv_freq was given");
  }
  p.k = at(a.ptr); p.v = at(b.ptr); p.k_cache = at(kc.ptr); p.v_cache = at(vc.ptr); p.page_table = s.table; p.q_start = s.start; p.kv_len = s.len; p.bad_pages = s.bad;
  p.dtype = a.dtype; p.tokens = a.n[0]; p.batch = s.size; p.kv_heads = a.n[1]; p.d = a.n[2]; p.num_pages = kc.n[0]; p.page_size = kc.n[1]; p.table_width = s.width;
  p.table_s0 = s.stride; p.k_st = a.s[0]; p.k_sh = a.s[1]; p.v_st = b.s[0]; p.v_sh = b.s[1];
  p.kc_sp = kc.s[0]; p.kc_sn = kc.s[1]; p.kc_sh = kc.s[2]; p.vc_sp = vc.s[0]; p.vc_sn = vc.s[1]; p.vc_sh = vc.s[2]; p.interleaved = interleaved;
  check(llc_cuda_kv_append(&p, streamOf(a.device)));
  if (given) wrote({kCache.ptr(), vCache.ptr(), qOut.ptr()});
  else wrote({kCache.ptr(), vCache.ptr()});
  return qOut;
}

py::object pagedAttention(py::handle q, py::handle kCache, py::handle vCache, py::handle table, py::handle start, py::handle len, py::object scale, int64_t window, int64_t sinks,
                          py::object maxQ, py::object out, py::handle bad) {
  Operand a = firstRows("q", q), kc = cacheOf("k_cache", kCache, a), vc = cacheOf("v_cache", vCache, a);
  sameShape(kc, vc);
  const int64_t kv = kc.n[2], d = kc.n[3];
  if (a.n[2] != d || a.n[1] == 0 || a.n[1] % kv) a.bad("expected [tokens, a multiple of " + std::to_string(kv) + ", " + std::to_string(d) + "], got " + a.shape());
  const Batch s = batchOf(table, start, len, bad, a.device);
  if (window < 0 || sinks < 0) throw py::value_error("window and sinks: must not be negative");
  const int64_t most = maxQ.is_none() ? a.n[0] : number("max_q", maxQ.ptr());
  if (most < 0) throw py::value_error("max_q: must not be negative");
  const bool given = !out.is_none();
  const Operand o = output("out", out, q, a);
  LlcPagedAttentionParams p{};
  p.q = at(a.ptr); p.k_cache = at(kc.ptr); p.v_cache = at(vc.ptr); p.out = at(o.ptr); p.page_table = s.table; p.q_start = s.start; p.kv_len = s.len; p.bad_pages = s.bad;
  p.dtype = a.dtype; p.scale = scale.is_none() ? (float)(1.0 / std::sqrt((double)d)) : (float)py::float_(scale);
  p.tokens = a.n[0]; p.batch = s.size; p.heads = a.n[1]; p.kv_heads = kv; p.d = d; p.max_q = most; p.num_pages = kc.n[0]; p.page_size = kc.n[1];
  p.table_width = s.width; p.table_s0 = s.stride; p.window = window; p.sinks = sinks;
  p.q_st = a.s[0]; p.q_sh = a.s[1]; p.o_st = o.s[0]; p.o_sh = o.s[1];
  p.kc_sp = kc.s[0]; p.kc_sn = kc.s[1]; p.kc_sh = kc.s[2]; p.vc_sp = vc.s[0]; p.vc_sn = vc.s[1]; p.vc_sh = vc.s[2];
  // scratch from the caching allocator at every call: ordered with the stream, and a captured graph gets memory of its own
  py::object scratch;
  if (const int64_t bytes = llc_cuda_paged_attention_workspace(&p)) {
    const Torch& t = torch();
    py::object n = got(PyLong_FromLongLong((bytes + 3) / 4)), dev = got(PyObject_GetAttr(q.ptr(), t.nDeviceOf));
    PyObject* const args[] = {n.ptr(), t.f32.ptr(), dev.ptr()};
    scratch = got(PyObject_Vectorcall(t.empty.ptr(), args, 1, t.kwEmpty));
    p.workspace = at(PyLong_AsUnsignedLongLong(got(PyObject_CallMethodNoArgs(scratch.ptr(), t.nPtr)).ptr()));
    p.workspace_bytes = bytes;
  }
  check(llc_cuda_paged_attention(&p, streamOf(a.device)));
  if (given) wrote({out.ptr()});
  return out;
}

// The three as plain functions of the interpreter (positional arguments, a fixed number of them): its own calling convention costs a tenth of
// a wrapped function's.  C++ exceptions end here.
template <Py_ssize_t N, typename F> PyObject* enter(const char* name, Py_ssize_t n, F f) {
  try {
    if (n != N) throw py::type_error(std::string(name) + ": expected " + std::to_string(N) + " arguments, got " + std::to_string(n));
    torch().look();
    return f().release().ptr();
  } catch (py::error_already_set& e) {
    e.restore();
  } catch (const py::builtin_exception& e) {
    e.set_error();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
py::object own(PyObject* o) { return py::reinterpret_borrow<py::object>(o); }
bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw py::error_already_set();
  return x != 0;
}
PyObject* rotaryEntry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return enter<6>("rotary", n, [&] { return rotary(a[0], a[1], a[2], a[3], truth(a[4]), own(a[5])); });
}
PyObject* kvAppendEntry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return enter<14>("kv_append", n, [&] { return kvAppend(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], truth(a[11]), own(a[12]), a[13]); });
}
PyObject* pagedEntry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return enter<12>("paged_attention", n, [&] {
    return pagedAttention(a[0], a[1], a[2], a[3], a[4], a[5], own(a[6]), number("window", a[7]), number("sinks", a[8]), own(a[9]), own(a[10]), a[11]);
  });
}
PyMethodDef kOps[] = {{"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&rotaryEntry)), METH_FASTCALL, nullptr},
                      {"kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&kvAppendEntry)), METH_FASTCALL, nullptr},
                      {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&pagedEntry)), METH_FASTCALL, nullptr}};

}  // namespace

PYBIND11_MODULE(llcompiler_, m) {
  m.doc() = "B200 execution backend with the llcompiler_ module surface";
  auto tensor = m.def_submodule("tensor");
  py::class_<Tensor>(tensor, "Tensor", py::buffer_protocol())
      .def(py::init<>())
      .def_buffer(&bufferOf)
      .def("to_numpy", [](Tensor& t) { return py::array(bufferOf(t)); })
      .def(py::init<uintptr_t, uintptr_t, int, int64_t, std::vector<int64_t>, std::vector<int64_t>, int>(), py::arg("data_ptr"), py::arg("base_ptr"),
           py::arg("type"), py::arg("offset"), py::arg("size"), py::arg("stride"), py::arg("device") = -1)
      .def_readwrite("data", &Tensor::data).def_readwrite("base", &Tensor::base).def_readwrite("offset", &Tensor::offset)
      .def_readwrite("size", &Tensor::size).def_readwrite("stride", &Tensor::stride).def_readwrite("type", &Tensor::type)
      .def_readwrite("device", &Tensor::device)
      .def("print", &Tensor::print);
  tensor.attr("INT8") = (int)LLC_INT8; tensor.attr("INT16") = (int)LLC_INT16; tensor.attr("INT32") = (int)LLC_INT32;
  tensor.attr("INT64") = (int)LLC_INT64; tensor.attr("FLOAT32") = (int)LLC_FLOAT32; tensor.attr("DOUBL64") = (int)LLC_FLOAT64;
  tensor.attr("INT1") = (int)LLC_INT1; tensor.attr("FLOAT16") = (int)LLC_FLOAT16; tensor.attr("BFLOAT16") = (int)LLC_BFLOAT16;

  auto compiler = m.def_submodule("compiler");
  py::class_<Compiler>(compiler, "Compiler")
      .def(py::init<>())
      .def("compile_mlir_to_shared_lib", &Compiler::compile_mlir_to_shared_lib)
      .def("run_pass", &Compiler::run_pass);
  py::class_<CompileOptions>(compiler, "CompileOptions")
      .def(py::init<>())
      .def("set_log_root", [](CompileOptions& o, const std::string& v) { o.log_root = v; })
      .def("set_mode", [](CompileOptions& o, const std::string& v) { o.mode = v; })
      .def("set_target", [](CompileOptions& o, const std::string& v) { o.target = v; })
      .def("set_log_level", [](CompileOptions& o, const std::string& v) { o.log_level = v; })
      .def("set_pipeline", [](CompileOptions& o, const std::string& v) { o.pipeline = v; })
      .def("set_global_layout", [](CompileOptions& o, const std::string& v) { o.global_layout = v; })
      .def("set_cpu", [](CompileOptions& o, const std::string& v) { o.cpu = v; })
      .def("set_mtriple", [](CompileOptions& o, const std::string& v) { o.mtriple = v; })
      .def("set_precision", [](CompileOptions& o, const std::string& v) { o.precision = v; })
      .def("display_llvm_passes", [](CompileOptions& o, bool v) { o.llvm_passes = v; })
      .def("display_mlir_passes", [](CompileOptions& o, bool v) { o.mlir_passes = v; });

  auto executor = m.def_submodule("executor");
  executor.def("get_tool", &getTool);
  py::class_<Execution>(executor, "Execution")
      .def(py::init<>())
      .def("load", &Execution::load, py::arg("path"), py::arg("device") = 0, py::arg("weight_dir") = "")
      .def("loaded_from_pool", &Execution::loaded_from_pool)
      .def("run", &Execution::run, py::arg("inputs"), py::arg("outs"), py::arg("stream") = 0)
      .def("run_with_symbols", &Execution::run_with_symbols, py::arg("symbols"), py::arg("inputs"), py::arg("outs"), py::arg("stream") = 0)
      .def("output_shapes", &Execution::output_shapes)
      .def("profile", &Execution::profile, py::arg("symbols"), py::arg("inputs"), py::arg("outs"), py::arg("reps") = 5, py::arg("stream") = 0)
      .def("status", &Execution::status)
      .def("num_inputs", &Execution::num_inputs).def("num_outputs", &Execution::num_outputs).def("num_symbols", &Execution::num_symbols)
      .def("last_launch_count", &Execution::last_launch_count).def("arena_bytes", &Execution::arena_bytes);
  auto ops = m.def_submodule("ops");
  for (PyMethodDef& f : kOps) ops.attr(f.ml_name) = got(PyCFunction_NewEx(&f, nullptr, nullptr));
  ops.def("status", []() { return llc_cuda_status(); }, py::call_guard<py::gil_scoped_release>());
  m.def("version", []() { return std::string(llc_version()); });
}
