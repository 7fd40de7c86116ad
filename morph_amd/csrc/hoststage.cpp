// The host side of the state space operators and of the 8-bit moments' values for tensors that need no preparation;
// see hostlayers.cpp.  In Python a norm of 8 rows took 18 us beside 3.2 on the device, a step of the scan 29 beside 13,
// the values of 200 tensors' moments 600 beside 16.
#include "hostcalls.h"

#include "../../include/morph_state_space.h"

namespace {

struct Calls {  // of the library, by address
  decltype(&morph_norm_forward) norm_forward;
  decltype(&morph_norm_workspace_bytes) norm_workspace_bytes;
  decltype(&morph_norm_backward) norm_backward;
  decltype(&morph_conv_forward) conv_forward;
  decltype(&morph_conv_workspace_bytes) conv_workspace_bytes;
  decltype(&morph_conv_backward) conv_backward;
  decltype(&morph_ssm_forward) ssm_forward;
  decltype(&morph_ssm_workspace_bytes) ssm_workspace_bytes;
  decltype(&morph_ssm_backward) ssm_backward;
  decltype(&morph_moment_decode) moment_decode;
};

const void* data(const at::Tensor* t) { return t != nullptr ? t->const_data_ptr() : nullptr; }
void* data(at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
py::object given(at::Tensor t) { return t.defined() ? wrap(std::move(t)) : py::object(py::none()); }

class StageCalls {
 public:
  explicit StageCalls(const std::vector<uint64_t>& a) {
    if (a.size() != 10) throw std::invalid_argument("ten entry points expected");
    c_.norm_forward = reinterpret_cast<decltype(c_.norm_forward)>(a[0]);
    c_.norm_workspace_bytes = reinterpret_cast<decltype(c_.norm_workspace_bytes)>(a[1]);
    c_.norm_backward = reinterpret_cast<decltype(c_.norm_backward)>(a[2]);
    c_.conv_forward = reinterpret_cast<decltype(c_.conv_forward)>(a[3]);
    c_.conv_workspace_bytes = reinterpret_cast<decltype(c_.conv_workspace_bytes)>(a[4]);
    c_.conv_backward = reinterpret_cast<decltype(c_.conv_backward)>(a[5]);
    c_.ssm_forward = reinterpret_cast<decltype(c_.ssm_forward)>(a[6]);
    c_.ssm_workspace_bytes = reinterpret_cast<decltype(c_.ssm_workspace_bytes)>(a[7]);
    c_.ssm_backward = reinterpret_cast<decltype(c_.ssm_backward)>(a[8]);
    c_.moment_decode = reinterpret_cast<decltype(c_.moment_decode)>(a[9]);
  }

  // y, or with `train` (y, stats).
  py::object norm_forward(py::handle ox, py::handle ow, py::handle ob, double eps, bool train) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ox);
    const at::Tensor* x = here.tensor(ox);
    morph_norm a;
    if (x == nullptr || !norm(here, *x, ow, ob, eps, a)) return py::none();
    at::Tensor y = here.empty(x->sizes(), x->scalar_type()), stats;
    if (train) stats = here.empty({2, a.rows}, at::kFloat);
    const int rc = released([&] {
      return c_.norm_forward(&a, code(x->scalar_type()), y.data_ptr(), static_cast<float*>(data(stats)), here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    if (!train) return wrap(std::move(y));
    return py::make_tuple(wrap(std::move(y)), wrap(std::move(stats)));
  }

  // (dx, dweight or None, dbias or None).
  py::object norm_backward(py::handle ody, py::handle ox, py::handle ow, py::handle ob, py::handle ostats,
                           double eps) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ody);
    const at::Tensor *dy = here.tensor(ody), *x = here.tensor(ox), *stats = here.tensor(ostats);
    morph_norm a;
    if (dy == nullptr || x == nullptr || stats == nullptr || !norm(here, *x, ow, ob, eps, a)) return py::none();
    if (dy->scalar_type() != x->scalar_type() || dy->sizes() != x->sizes() || !dy->is_contiguous() ||
        !holds(*stats, at::kFloat, 2 * a.rows))
      return py::none();
    at::Tensor dx = here.empty(x->sizes(), x->scalar_type()), dw, db, workspace;
    const at::ScalarType type = a.weight_dtype == MORPH_DTYPE_F32 ? at::kFloat : x->scalar_type();
    if (a.weight != nullptr) dw = here.empty({a.cols}, type);
    if (a.bias != nullptr) db = here.empty({a.cols}, type);
    const size_t size = a.weight != nullptr || a.bias != nullptr ? c_.norm_workspace_bytes(a.rows, a.cols) : 0;
    if (size > 0) workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.norm_backward(&a, code(x->scalar_type()), stats->const_data_ptr<float>(), dy->const_data_ptr(), a.cols,
                              dx.data_ptr(), data(dw), data(db), data(workspace), size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(dx)), given(std::move(dw)), given(std::move(db)));
  }

  // (u, the last inputs).
  py::object conv_forward(py::handle ox, py::handle ow, py::handle ob, py::handle os) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ox);
    morph_conv a;
    at::ScalarType type;
    if (!conv(here, ox, ow, ob, os, a, type)) return py::none();
    at::Tensor u = here.empty({a.batch, a.steps, a.dim}, type), last = here.empty({a.batch, a.taps - 1, a.dim}, type);
    const int rc = released([&] { return c_.conv_forward(&a, code(type), u.data_ptr(), last.data_ptr(), here.stream()); });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(u)), wrap(std::move(last)));
  }

  // (dx, dweight, dbias or None, dstate).
  py::object conv_backward(py::handle odu, py::handle ox, py::handle ow, py::handle ob, py::handle os,
                           py::handle odlast) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(odu);
    morph_conv a;
    at::ScalarType type;
    const at::Tensor *du = here.tensor(odu), *dlast = nullptr;
    if (du == nullptr || !conv(here, ox, ow, ob, os, a, type) || !sequence(*du, type, a.batch, a.steps, a.dim)) return py::none();
    if (!optional(here, odlast, type, {a.batch, a.taps - 1, a.dim}, dlast)) return py::none();
    const at::ScalarType wtype = a.weight_dtype == MORPH_DTYPE_F32 ? at::kFloat : type;
    at::Tensor dx = here.empty({a.batch, a.steps, a.dim}, type), dw = here.empty({a.dim, a.taps}, wtype), db, workspace;
    at::Tensor dstate = here.empty({a.batch, a.taps - 1, a.dim}, type);
    if (a.bias != nullptr) db = here.empty({a.dim}, wtype);
    const size_t size = c_.conv_workspace_bytes(a.batch, a.steps, a.dim, a.taps);
    if (size > 0) workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.conv_backward(&a, code(type), du->const_data_ptr(), du->stride(0), du->stride(1), data(dlast), dx.data_ptr(),
                              dw.data_ptr(), data(db), dstate.data_ptr(), data(workspace), size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(dx)), wrap(std::move(dw)), given(std::move(db)), wrap(std::move(dstate)));
  }

  // (y, last), and with `train` the kept states.  inputs: x, dt, A, B, C, skip, z, dt_bias, state.
  py::object ssm_forward(const py::tuple& inputs, bool train) const {
    if (c10::impl::dispatch_mode_enabled() || inputs.size() != 9) return py::none();
    const Here here(inputs[0]);
    morph_ssm a;
    at::ScalarType type;
    if (!ssm(here, inputs, a, type)) return py::none();
    at::Tensor y = here.empty({a.batch, a.steps, a.dim}, type), last = here.empty({a.batch, a.dim, a.states}, at::kFloat);
    at::Tensor kept, workspace;
    if (train) kept = here.empty({a.batch, spans(a.steps), a.dim, a.states}, at::kFloat);
    const size_t size = c_.ssm_workspace_bytes(a.batch, a.steps, a.dim, a.states, 0);
    if (size > 0) workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.ssm_forward(&a, code(type), y.data_ptr(), static_cast<float*>(last.data_ptr()),
                            static_cast<float*>(data(kept)), data(workspace), size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    if (!train) return py::make_tuple(wrap(std::move(y)), wrap(std::move(last)));
    return py::make_tuple(wrap(std::move(y)), wrap(std::move(last)), wrap(std::move(kept)));
  }

  // The gradients of the inputs, in their order (the state's always).
  py::object ssm_backward(py::handle ody, const py::tuple& inputs, py::handle okept, py::handle odlast) const {
    if (c10::impl::dispatch_mode_enabled() || inputs.size() != 9) return py::none();
    const Here here(ody);
    morph_ssm a;
    at::ScalarType type;
    const at::Tensor *dy = here.tensor(ody), *kept = here.tensor(okept), *dlast = nullptr;
    if (dy == nullptr || kept == nullptr || !ssm(here, inputs, a, type) ||
        !sequence(*dy, type, a.batch, a.steps, a.dim) || dy->stride(1) > MORPH_SSM_MAX_STEP ||
        !holds(*kept, at::kFloat, a.batch * spans(a.steps) * a.dim * a.states) ||
        !optional(here, odlast, at::kFloat, {a.batch, a.dim, a.states}, dlast))
      return py::none();
    const int64_t shape[3] = {a.batch, a.steps, a.dim}, small[3] = {a.batch, a.steps, a.states};
    at::Tensor dx = here.empty(shape, type), ddt = here.empty(shape, type), dz, dB = here.empty(small, type);
    at::Tensor dC = here.empty(small, type), dA = here.empty({a.dim, a.states}, at::kFloat), dskip, ddt_bias;
    at::Tensor dfirst = here.empty({a.batch, a.dim, a.states}, at::kFloat);
    if (a.z != nullptr) dz = here.empty(shape, type);
    if (a.skip != nullptr) dskip = here.empty({a.dim}, at::kFloat);
    if (a.dt_bias != nullptr) ddt_bias = here.empty({a.dim}, at::kFloat);
    const morph_ssm_grads g{data(dx), data(ddt), data(dz), data(dB), data(dC), static_cast<float*>(data(dA)),
                            static_cast<float*>(data(dskip)), static_cast<float*>(data(ddt_bias)),
                            static_cast<float*>(data(dfirst))};
    const size_t size = c_.ssm_workspace_bytes(a.batch, a.steps, a.dim, a.states, 1);
    at::Tensor workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.ssm_backward(&a, code(type), kept->const_data_ptr<float>(), dy->const_data_ptr(), dy->stride(0),
                             dy->stride(1), dlast != nullptr ? dlast->const_data_ptr<float>() : nullptr, &g,
                             workspace.data_ptr(), size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(dx)), wrap(std::move(ddt)), wrap(std::move(dA)), wrap(std::move(dB)),
                          wrap(std::move(dC)), given(std::move(dskip)), given(std::move(dz)), given(std::move(ddt_bias)),
                          wrap(std::move(dfirst)));
  }

  // The values of an optimizer's 8-bit moments into `out`, a list of a pair a parameter: True, or None where
  // anything is not as expected.  groups, state: the optimizer's.
  py::object moments(py::handle groups, py::handle state, py::handle out, py::handle first) const {
    if (c10::impl::dispatch_mode_enabled() || !PyList_CheckExact(groups.ptr()) || !PyDict_Check(state.ptr()) ||
        !PyList_CheckExact(out.ptr()))
      return py::none();
    const Here here(first);
    std::vector<morph_moment_values> values;
    at::ScalarType type = at::kByte;
    Py_ssize_t i = 0, in_state = 0;
    static PyObject* const params = PyUnicode_InternFromString("params");
    static PyObject* const names[2] = {PyUnicode_InternFromString("exp_avg"), PyUnicode_InternFromString("exp_avg_sq")};
    for (Py_ssize_t g = 0; g < PyList_GET_SIZE(groups.ptr()); ++g) {
      PyObject* group = PyList_GET_ITEM(groups.ptr(), g);
      PyObject* list = PyDict_CheckExact(group) ? PyDict_GetItemWithError(group, params) : nullptr;
      if (list == nullptr || !PyList_CheckExact(list)) return py::none();
      for (Py_ssize_t j = 0; j < PyList_GET_SIZE(list); ++j, ++i) {
        PyObject* po = PyList_GET_ITEM(list, j);
        const at::Tensor* p = here.tensor(po);
        PyObject *owner = nullptr, *held = nullptr;  // in the parameters' order: a lookup by them takes longer
        if (p == nullptr || !PyDict_Next(state.ptr(), &in_state, &owner, &held) || owner != po || !PyDict_Check(held) ||
            i >= PyList_GET_SIZE(out.ptr()))
          return py::none();
        PyObject* pair = PyList_GET_ITEM(out.ptr(), i);
        if (!PyTuple_CheckExact(pair) || PyTuple_GET_SIZE(pair) != 2) return py::none();
        const int64_t n = p->numel();
        const void* from[2];
        void* to[2];
        for (int k = 0; k < 2; ++k) {
          PyObject* om = PyDict_GetItemWithError(held, names[k]);
          const at::Tensor *m = om != nullptr ? here.tensor(om) : nullptr, *o = here.tensor(PyTuple_GET_ITEM(pair, k));
          if (m == nullptr || o == nullptr || !holds(*m, at::kByte, (n + MORPH_MOMENT_GROUP - 1) / MORPH_MOMENT_GROUP * (MORPH_MOMENT_GROUP + 1)))
            return py::none();
          if (type == at::kByte) type = o->scalar_type();
          if (code(type) < 0 || !holds(*o, type, n)) return py::none();
          from[k] = m->const_data_ptr(), to[k] = o->data_ptr();
        }
        if (n > 0) values.push_back(morph_moment_values{from[0], from[1], to[0], to[1], n});
      }
    }
    if (PyErr_Occurred()) throw py::error_already_set();
    if (i != PyList_GET_SIZE(out.ptr()) || i == 0) return py::none();
    const int rc = released([&] { return c_.moment_decode(values.data(), (int)values.size(), code(type), here.stream()); });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::bool_(true);
  }

 private:
  Calls c_;

  static int64_t spans(int64_t steps) { return (steps + MORPH_SSM_SPAN - 1) / MORPH_SSM_SPAN; }

  // None, or a contiguous tensor of this type and shape.
  static bool optional(const Here& here, py::handle o, at::ScalarType type, std::initializer_list<int64_t> shape,
                       const at::Tensor*& t) {
    t = nullptr;
    if (o.is_none()) return true;
    t = here.tensor(o);
    return t != nullptr && t->scalar_type() == type && t->sizes() == at::IntArrayRef(shape) && t->is_contiguous();
  }

  static bool sequence(const at::Tensor& t, at::ScalarType type, int64_t batch, int64_t steps, int64_t dim) {
    return t.dim() == 3 && t.scalar_type() == type && t.size(0) == batch && t.size(1) == steps && t.size(2) == dim &&
           (dim == 1 || t.stride(2) == 1);
  }

  // A weight and a bias of x's type or FP32, one of them at least there or FP32 for none.
  static bool weights(const Here& here, at::ScalarType type, py::handle ow, py::handle ob, int64_t n, const at::Tensor*& w,
                      const at::Tensor*& b, int32_t& dtype) {
    at::ScalarType wtype = at::kFloat;
    for (py::handle o : {ow, ob}) {
      if (o.is_none()) continue;
      const at::Tensor* t = here.tensor(o);
      if (t == nullptr) return false;
      wtype = t->scalar_type();
      break;
    }
    if (wtype != at::kFloat && wtype != type) return false;
    dtype = code(wtype);
    return optional(here, ow, wtype, {n}, w) && optional(here, ob, wtype, {n}, b);
  }

  static bool norm(const Here& here, const at::Tensor& x, py::handle ow, py::handle ob, double eps, morph_norm& a) {
    if (x.dim() == 0 || code(x.scalar_type()) < 0 || x.numel() == 0 || !(eps >= 0 && eps < INFINITY)) return false;
    a.cols = x.size(-1), a.rows = x.numel() / a.cols, a.x_ld = a.cols;
    if (!x.is_contiguous()) {
      a.x_ld = x.dim() == 2 ? rows_of(x, x.scalar_type(), a.rows, a.cols) : 0;
      if (a.x_ld == 0) return false;
    }
    const at::Tensor *w, *b;
    if (!weights(here, x.scalar_type(), ow, ob, a.cols, w, b, a.weight_dtype)) return false;
    a.x = x.const_data_ptr(), a.weight = data(w), a.bias = data(b), a.eps = (float)eps;
    return true;
  }

  static bool conv(const Here& here, py::handle ox, py::handle ow, py::handle ob, py::handle os, morph_conv& a,
                   at::ScalarType& type) {
    const at::Tensor *x = here.tensor(ox), *w = here.tensor(ow), *b, *s;
    if (x == nullptr || w == nullptr || x->dim() != 3 || code(x->scalar_type()) < 0 || x->numel() == 0 || w->dim() != 2)
      return false;
    type = x->scalar_type();
    const at::ScalarType wtype = w->scalar_type();
    a.batch = x->size(0), a.steps = x->size(1), a.dim = x->size(2), a.taps = (int32_t)w->size(1);
    if (!sequence(*x, type, a.batch, a.steps, a.dim) || (wtype != at::kFloat && wtype != type) || w->size(0) != a.dim ||
        w->size(1) < 2 || w->size(1) > MORPH_CONV_MAX_TAPS || !w->is_contiguous())
      return false;
    if (!optional(here, ob, wtype, {a.dim}, b) || !optional(here, os, type, {a.batch, a.taps - 1, a.dim}, s)) return false;
    a.x = x->const_data_ptr(), a.before = data(s), a.weight = w->const_data_ptr(), a.bias = data(b);
    a.x_batch = x->stride(0), a.x_step = x->stride(1), a.weight_dtype = code(wtype);
    return true;
  }

  static bool ssm(const Here& here, const py::tuple& in, morph_ssm& a, at::ScalarType& type) {
    const at::Tensor *x = here.tensor(in[0]), *dt = here.tensor(in[1]), *A = here.tensor(in[2]), *B = here.tensor(in[3]),
                     *C = here.tensor(in[4]), *z = nullptr, *skip, *bias, *first;
    if (x == nullptr || dt == nullptr || A == nullptr || B == nullptr || C == nullptr || x->dim() != 3 ||
        code(x->scalar_type()) < 0 || x->numel() == 0 || A->dim() != 2)
      return false;
    type = x->scalar_type();
    a = morph_ssm{};
    a.batch = x->size(0), a.steps = x->size(1), a.dim = x->size(2);
    if (A->size(1) < 1 || A->size(1) > MORPH_SSM_MAX_STATES || !holds(*A, at::kFloat, a.dim * A->size(1)) || A->size(0) != a.dim)
      return false;
    a.states = (int32_t)A->size(1);
    if (!in[6].is_none()) {
      z = here.tensor(in[6]);
      if (z == nullptr || !sequence(*z, type, a.batch, a.steps, a.dim)) return false;
    }
    if (!sequence(*x, type, a.batch, a.steps, a.dim) || !sequence(*dt, type, a.batch, a.steps, a.dim) ||
        !sequence(*B, type, a.batch, a.steps, a.states) || !sequence(*C, type, a.batch, a.steps, a.states) ||
        !optional(here, in[5], at::kFloat, {a.dim}, skip) || !optional(here, in[7], at::kFloat, {a.dim}, bias) ||
        !optional(here, in[8], at::kFloat, {a.batch, a.dim, a.states}, first))
      return false;
    for (const at::Tensor* t : {x, dt, B, C, z})
      if (t != nullptr && t->stride(1) > MORPH_SSM_MAX_STEP) return false;
    a.x = data(x), a.dt = data(dt), a.z = data(z), a.B = data(B), a.C = data(C);
    a.A = static_cast<const float*>(data(A)), a.skip = static_cast<const float*>(data(skip));
    a.dt_bias = static_cast<const float*>(data(bias)), a.first = static_cast<const float*>(data(first));
    a.x_batch = x->stride(0), a.x_step = x->stride(1), a.dt_batch = dt->stride(0), a.dt_step = dt->stride(1);
    if (z != nullptr) a.z_batch = z->stride(0), a.z_step = z->stride(1);
    a.B_batch = B->stride(0), a.B_step = B->stride(1), a.C_batch = C->stride(0), a.C_step = C->stride(1);
    return true;
  }
};

}  // namespace

void bind_stage(py::module_& m) {
  py::class_<StageCalls>(m, "StageCalls")
      .def(py::init<const std::vector<uint64_t>&>())
      .def("norm_forward", &StageCalls::norm_forward)
      .def("norm_backward", &StageCalls::norm_backward)
      .def("conv_forward", &StageCalls::conv_forward)
      .def("conv_backward", &StageCalls::conv_backward)
      .def("ssm_forward", &StageCalls::ssm_forward)
      .def("ssm_backward", &StageCalls::ssm_backward)
      .def("moments", &StageCalls::moments);
}
