// The host side of the layer operators for tensors that need no preparation: the checks, the
// outputs and the launches of a call in one native call.
//
// For one token or a small batch the host is what a call takes: a step of the recurrence ran 3 us
// on the device and 21 us in Python, a pack and an unpack of 96 x 200 values 6 and 26.
//
// Every method returns None for anything that it does not recognise (no plain tensor on the
// current device, another type, a layout that needs a copy, shapes that do not fit); the
// caller then takes the Python path, which prepares it or raises.  A status of the library
// comes back as an int.
#include "hostcalls.h"

namespace {

struct Calls {  // of the library, by address
  decltype(&morph_act_pack) act_pack;
  decltype(&morph_act_unpack) act_unpack;
  decltype(&morph_ffn_workspace_bytes) ffn_workspace_bytes;
  decltype(&morph_ffn_forward) ffn_forward;
  decltype(&morph_ffn_backward) ffn_backward;
  decltype(&morph_scan_workspace_bytes) scan_workspace_bytes;
  decltype(&morph_scan_forward) scan_forward;
  decltype(&morph_scan_backward) scan_backward;
};

bool half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int64_t groups_of(int64_t n) { return (n + MORPH_ACT_GROUP - 1) / MORPH_ACT_GROUP; }

class LayerCalls {
 public:
  explicit LayerCalls(const std::vector<uint64_t>& a) {
    if (a.size() != 8) throw std::invalid_argument("eight entry points expected");
    c_.act_pack = reinterpret_cast<decltype(c_.act_pack)>(a[0]);
    c_.act_unpack = reinterpret_cast<decltype(c_.act_unpack)>(a[1]);
    c_.ffn_workspace_bytes = reinterpret_cast<decltype(c_.ffn_workspace_bytes)>(a[2]);
    c_.ffn_forward = reinterpret_cast<decltype(c_.ffn_forward)>(a[3]);
    c_.ffn_backward = reinterpret_cast<decltype(c_.ffn_backward)>(a[4]);
    c_.scan_workspace_bytes = reinterpret_cast<decltype(c_.scan_workspace_bytes)>(a[5]);
    c_.scan_forward = reinterpret_cast<decltype(c_.scan_forward)>(a[6]);
    c_.scan_backward = reinterpret_cast<decltype(c_.scan_backward)>(a[7]);
  }

  // (codes, exponents) of x.
  py::object pack(py::handle ox) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ox);
    const at::Tensor* x = here.tensor(ox);
    if (x == nullptr || x->dim() == 0 || code(x->scalar_type()) < 0 || !x->is_contiguous() || x->numel() == 0)
      return py::none();
    const int64_t cols = x->size(-1), rows = x->numel() / cols, groups = groups_of(cols);
    at::Tensor codes = here.empty({rows, groups * MORPH_ACT_GROUP}, at::kByte);
    at::Tensor exps = here.empty({rows, groups}, at::kByte);
    const int rc = released([&] {
      return c_.act_pack(x->const_data_ptr(), code(x->scalar_type()), rows, cols, cols, bytes(codes), bytes(exps),
                         here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(codes)), wrap(std::move(exps)));
  }

  // What codes and exponents of a [.., cols] activation stand for, in the type of this dtype code (with
  // MORPH_ACT_SATURATE or without).
  py::object unpack(py::handle ocodes, py::handle oexps, const std::vector<int64_t>& shape, int dtype) const {
    if (c10::impl::dispatch_mode_enabled() || shape.empty() || dtype < 0) return py::none();
    const Here here(ocodes);
    const at::Tensor *codes = here.tensor(ocodes), *exps = here.tensor(oexps);
    if (codes == nullptr || exps == nullptr) return py::none();
    const int64_t cols = shape.back(), groups = groups_of(cols);
    int64_t n = 1;
    for (int64_t s : shape) n *= s;
    if (n == 0) return py::none();
    const int64_t rows = n / cols;
    auto fits = [&](const at::Tensor& t, int64_t width) {
      return t.scalar_type() == at::kByte && t.dim() == 2 && t.size(0) == rows && t.size(1) == width &&
             t.is_contiguous();
    };
    if (!fits(*codes, groups * MORPH_ACT_GROUP) || !fits(*exps, groups)) return py::none();
    const int type = dtype & ~MORPH_ACT_SATURATE;
    at::Tensor out = here.empty(shape, type == MORPH_DTYPE_F32 ? at::kFloat : type == MORPH_DTYPE_F16 ? at::kHalf : at::kBFloat16);
    const int rc = released([&] {
      return c_.act_unpack(codes->const_data_ptr<uint8_t>(), exps->const_data_ptr<uint8_t>(), rows, cols,
                           out.data_ptr(), dtype, cols, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return wrap(std::move(out));
  }

  // (y,) and behind it what `keep` says: the projections [2, rows, 32 G], or codes and exponents
  // of x, of the gate's and of the up projection.
  py::object ffn_forward(py::handle ox, py::handle og, py::handle ou, py::handle od, int keep) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ox);
    const at::Tensor *x = here.tensor(ox), *gate = here.tensor(og), *up = here.tensor(ou), *down = here.tensor(od);
    morph_ffn block;
    if (x == nullptr || !x->is_contiguous() || x->numel() == 0 || !weights(*x, gate, up, down, block)) return py::none();
    block.x = x->const_data_ptr(), block.x_ld = block.d;
    const int64_t rows = block.rows, groups = groups_of(block.ff), wide = groups * MORPH_ACT_GROUP;
    at::Tensor y = here.empty(x->sizes(), x->scalar_type());
    morph_ffn_saved saved{};
    saved.keep = keep;
    py::list out;
    if (keep == MORPH_FFN_KEEP_FULL) {
      at::Tensor kept = here.empty({2, rows, wide}, at::kFloat);
      saved.gate = kept.data_ptr();
      saved.up = static_cast<float*>(saved.gate) + rows * wide;
      out.append(wrap(std::move(kept)));
    } else if (keep == MORPH_FFN_KEEP_ACT8) {
      auto make = [&](int64_t width) {
        at::Tensor t = here.empty({rows, width}, at::kByte);
        uint8_t* p = bytes(t);
        out.append(wrap(std::move(t)));
        return p;
      };
      saved.x_codes = make(groups_of(block.d) * MORPH_ACT_GROUP);
      saved.x_exponents = make(groups_of(block.d));
      saved.gate = make(wide);
      saved.gate_exponents = make(groups);
      saved.up = make(wide);
      saved.up_exponents = make(groups);
    } else if (keep != MORPH_FFN_KEEP_NONE) {
      return py::none();
    }
    const size_t size = c_.ffn_workspace_bytes(rows, block.d, block.ff, keep, 0);
    const at::Tensor workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.ffn_forward(&block, code(x->scalar_type()), keep == MORPH_FFN_KEEP_NONE ? nullptr : &saved,
                            y.data_ptr(), block.d, workspace.data_ptr(), size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    if (keep == MORPH_FFN_KEEP_NONE) return wrap(std::move(y));
    return py::make_tuple(wrap(std::move(y)), out);
  }

  // (dx, dgate, dup, ddown); kept: (x, projections) or the six byte tensors of ffn_forward.
  py::object ffn_backward(py::handle ody, const py::tuple& kept, py::handle og, py::handle ou, py::handle od,
                          int keep) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ody);
    const at::Tensor *dy = here.tensor(ody), *gate = here.tensor(og), *up = here.tensor(ou), *down = here.tensor(od);
    morph_ffn block;
    if (dy == nullptr || !dy->is_contiguous() || dy->numel() == 0 || !weights(*dy, gate, up, down, block))
      return py::none();
    block.x = nullptr, block.x_ld = block.d;
    const int64_t rows = block.rows, groups = groups_of(block.ff), wide = groups * MORPH_ACT_GROUP;
    morph_ffn_saved saved{};
    saved.keep = keep;
    if (keep == MORPH_FFN_KEEP_FULL && kept.size() == 2) {
      const at::Tensor *x = here.tensor(kept[0]), *p = here.tensor(kept[1]);
      if (x == nullptr || p == nullptr || !holds(*p, at::kFloat, 2 * rows * wide)) return py::none();
      block.x_ld = rows_of(*x, dy->scalar_type(), rows, block.d);
      if (block.x_ld == 0) return py::none();
      block.x = x->const_data_ptr();
      saved.gate = p->data_ptr();
      saved.up = static_cast<float*>(saved.gate) + rows * wide;
    } else if (keep == MORPH_FFN_KEEP_ACT8 && kept.size() == 6) {
      const int64_t gx = groups_of(block.d);
      const int64_t widths[6] = {gx * MORPH_ACT_GROUP, gx, wide, groups, wide, groups};
      uint8_t* p[6];
      for (int i = 0; i < 6; ++i) {
        const at::Tensor* t = here.tensor(kept[i]);
        if (t == nullptr || !holds(*t, at::kByte, rows * widths[i])) return py::none();
        p[i] = bytes(*t);
      }
      saved.x_codes = p[0], saved.x_exponents = p[1], saved.gate = p[2], saved.gate_exponents = p[3];
      saved.up = p[4], saved.up_exponents = p[5];
    } else {
      return py::none();
    }
    const at::ScalarType type = dy->scalar_type();
    at::Tensor dx = here.empty(dy->sizes(), type), dgate = here.empty({block.ff, block.d}, type);
    at::Tensor dup = here.empty({block.ff, block.d}, type), ddown = here.empty({block.d, block.ff}, type);
    const size_t size = c_.ffn_workspace_bytes(rows, block.d, block.ff, keep, 1);
    const at::Tensor workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.ffn_backward(&block, code(type), &saved, dy->const_data_ptr(), block.d, dx.data_ptr(),
                             dgate.data_ptr(), dup.data_ptr(), ddown.data_ptr(), workspace.data_ptr(), size,
                             here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(dx)), wrap(std::move(dgate)), wrap(std::move(dup)), wrap(std::move(ddown)));
  }

  // (y, last), and with `train` the kept states.
  py::object scan_forward(py::handle of, py::handle ov, py::handle oz, py::handle os, bool train) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(of);
    morph_scan a;
    at::ScalarType type;
    if (!scan(here, of, ov, oz, os, a, type)) return py::none();
    at::Tensor y = here.empty({a.batch, a.steps, a.dim}, type), last = here.empty({a.batch, a.dim}, at::kFloat);
    at::Tensor states;
    if (train) states = here.empty({a.batch, (a.steps + MORPH_SCAN_SPAN - 1) / MORPH_SCAN_SPAN, a.dim}, at::kFloat);
    const size_t size = c_.scan_workspace_bytes(a.batch, a.steps, a.dim, code(type), 0);
    at::Tensor workspace;
    if (size > 0) workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.scan_forward(&a, code(type), y.data_ptr(), static_cast<float*>(last.data_ptr()),
                             train ? static_cast<float*>(states.data_ptr()) : nullptr,
                             size > 0 ? workspace.data_ptr() : nullptr, size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    if (!train) return py::make_tuple(wrap(std::move(y)), wrap(std::move(last)));
    return py::make_tuple(wrap(std::move(y)), wrap(std::move(last)), wrap(std::move(states)));
  }

  // (df, dv, dz or None, ds0).
  py::object scan_backward(py::handle ody, py::handle of, py::handle ov, py::handle oz, py::handle os,
                           py::handle ostates, py::handle odlast) const {
    if (c10::impl::dispatch_mode_enabled()) return py::none();
    const Here here(ody);
    morph_scan a;
    at::ScalarType type;
    if (!scan(here, of, ov, oz, os, a, type)) return py::none();
    const at::Tensor *dy = here.tensor(ody), *states = here.tensor(ostates);
    if (dy == nullptr || states == nullptr || !sequence(*dy, type, a)) return py::none();
    if (!holds(*states, at::kFloat, a.batch * ((a.steps + MORPH_SCAN_SPAN - 1) / MORPH_SCAN_SPAN) * a.dim))
      return py::none();
    const float* dlast = nullptr;
    if (!odlast.is_none()) {
      const at::Tensor* t = here.tensor(odlast);
      if (t == nullptr || t->dim() != 2 || t->size(0) != a.batch || !holds(*t, at::kFloat, a.batch * a.dim))
        return py::none();
      dlast = t->const_data_ptr<float>();
    }
    const int64_t shape[3] = {a.batch, a.steps, a.dim};
    at::Tensor df = here.empty(shape, type), dv = here.empty(shape, type), dz;
    if (a.z != nullptr) dz = here.empty(shape, type);
    at::Tensor ds0 = here.empty({a.batch, a.dim}, at::kFloat);
    const size_t size = c_.scan_workspace_bytes(a.batch, a.steps, a.dim, code(type), 1);
    at::Tensor workspace;
    if (size > 0) workspace = here.empty({(int64_t)size}, at::kByte);
    const int rc = released([&] {
      return c_.scan_backward(&a, code(type), states->const_data_ptr<float>(), dy->const_data_ptr(), dy->stride(0),
                              dy->stride(1), dlast, df.data_ptr(), dv.data_ptr(),
                              a.z != nullptr ? dz.data_ptr() : nullptr, static_cast<float*>(ds0.data_ptr()),
                              size > 0 ? workspace.data_ptr() : nullptr, size, here.stream());
    });
    if (rc != MORPH_OK) return py::int_(rc);
    return py::make_tuple(wrap(std::move(df)), wrap(std::move(dv)), a.z != nullptr ? wrap(std::move(dz)) : py::object(py::none()),
                          wrap(std::move(ds0)));
  }

 private:
  Calls c_;

  static uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

  // The weights of a block for x (or dy) of [.., d], into `block`.
  static bool weights(const at::Tensor& x, const at::Tensor* gate, const at::Tensor* up, const at::Tensor* down,
                      morph_ffn& block) {
    if (gate == nullptr || up == nullptr || down == nullptr || x.dim() == 0 || !half(x.scalar_type()) ||
        gate->dim() != 2)
      return false;
    const at::ScalarType type = x.scalar_type();
    block.d = x.size(-1), block.ff = gate->size(0);
    if (block.d < 1 || block.ff < 1) return false;
    block.rows = x.numel() / block.d;
    block.gate_ld = rows_of(*gate, type, block.ff, block.d);
    block.up_ld = rows_of(*up, type, block.ff, block.d);
    block.down_ld = rows_of(*down, type, block.d, block.ff);
    block.gate = gate->const_data_ptr(), block.up = up->const_data_ptr(), block.down = down->const_data_ptr();
    return block.gate_ld > 0 && block.up_ld > 0 && block.down_ld > 0;
  }

  static bool sequence(const at::Tensor& t, at::ScalarType type, const morph_scan& a) {
    return t.dim() == 3 && t.scalar_type() == type && t.size(0) == a.batch && t.size(1) == a.steps &&
           t.size(2) == a.dim && (a.dim == 1 || t.stride(2) == 1);
  }

  static bool scan(const Here& here, py::handle of, py::handle ov, py::handle oz, py::handle os, morph_scan& a,
                   at::ScalarType& type) {
    const at::Tensor *f = here.tensor(of), *v = here.tensor(ov);
    if (f == nullptr || v == nullptr || f->dim() != 3 || code(f->scalar_type()) < 0 || f->numel() == 0) return false;
    type = f->scalar_type();
    a = morph_scan{};
    a.batch = f->size(0), a.steps = f->size(1), a.dim = f->size(2);
    if (!sequence(*f, type, a) || !sequence(*v, type, a)) return false;
    a.f = f->const_data_ptr(), a.f_batch = f->stride(0), a.f_step = f->stride(1);
    a.v = v->const_data_ptr(), a.v_batch = v->stride(0), a.v_step = v->stride(1);
    if (!oz.is_none()) {
      const at::Tensor* z = here.tensor(oz);
      if (z == nullptr || !sequence(*z, type, a)) return false;
      a.z = z->const_data_ptr(), a.z_batch = z->stride(0), a.z_step = z->stride(1);
    }
    if (!os.is_none()) {
      const at::Tensor* s = here.tensor(os);
      if (s == nullptr || s->dim() != 2 || s->size(0) != a.batch || !holds(*s, at::kFloat, a.batch * a.dim))
        return false;
      a.s0 = s->const_data_ptr<float>();
    }
    return true;
  }
};

}  // namespace

void bind_layers(py::module_& m) {
  py::class_<LayerCalls>(m, "LayerCalls")
      .def(py::init<const std::vector<uint64_t>&>())
      .def("pack", &LayerCalls::pack)
      .def("unpack", &LayerCalls::unpack)
      .def("ffn_forward", &LayerCalls::ffn_forward)
      .def("ffn_backward", &LayerCalls::ffn_backward)
      .def("scan_forward", &LayerCalls::scan_forward)
      .def("scan_backward", &LayerCalls::scan_backward);
}
