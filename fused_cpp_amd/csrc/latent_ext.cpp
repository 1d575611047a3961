// latent_ext.cpp -- the latent-attention operators of `fused_cpp_amd._moe_C`.
//
// Validates tensors (dtypes and shapes first, then devices, so that every
// refusal but the last can be reached without a GPU), makes rows start where
// the kernels' 16-byte loads need them, allocates outputs and workspaces from
// the torch caching allocator on the current stream of the tensors' device and
// calls the C ABI of libfcmoe.so.
#include <c10/core/DeviceGuard.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/fcmoe.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == FCMOE_OK, what, " failed: ", fcmoe_last_error()); }

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_dtype(const at::Tensor& t, at::ScalarType want, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == want, name, " must be ", want, ", got ", t.scalar_type());
}

void check_dim(const at::Tensor& t, int64_t dim, const char* name, const char* shape) {
  TORCH_CHECK_VALUE(t.dim() == dim, name, " must be ", shape, ", got ", t.sizes());
}

void check_index(const at::Tensor& t, int64_t size, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name, " must be int32 or int64, got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == size, name, " must be [", size, "], got ", t.sizes());
}

// Inference operators: a result that silently has no gradient, or no tangent
// of forward-mode differentiation, is refused.
bool has_tangent(const at::Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t.defined() && t._fw_grad(0).defined();
}
void check_no_grad(std::initializer_list<const at::Tensor*> ts, const char* what) {
  for (const at::Tensor* t : ts) {
    TORCH_CHECK(!c10::GradMode::is_enabled() || !t->defined() || !t->requires_grad(), what,
                ": inputs that require a gradient are not supported (use torch.no_grad())");
    TORCH_CHECK(!has_tangent(*t), what, ": inputs with a forward-mode tangent are not supported");
  }
}
// A tensor that a kernel wrote to: a graph that saved it before finds out.
void was_written(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_devices(const at::Tensor& first, std::initializer_list<const at::Tensor*> ts, const char* what) {
  TORCH_CHECK_VALUE(first.is_cuda(), what, ": tensors must be on the ROCm device, got ", first.device());
  for (const at::Tensor* t : ts)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == first.device(), what, ": tensors must share one device, got ",
                      t->device(), " and ", first.device());
}

at::Tensor opt(const OptTensor& t) { return has(t) ? *t : at::Tensor(); }

// Whether rows can be read or written in place: last dimension contiguous, the
// others' strides and the start at multiples of `unit` elements.
bool rows_ok(const at::Tensor& t, int64_t unit) {
  if (t.dim() == 0) return false;
  if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) % unit != 0) return false;
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % (unit * t.element_size()) == 0;
}
at::Tensor rows_for(const at::Tensor& t, int64_t unit) {
  if (rows_ok(t, unit)) return t;
  at::Tensor c = t.contiguous();
  return rows_ok(c, unit) ? c : c.clone();
}
// The stride of a dimension of one entry is not used; torch may report any.
int64_t stride_at(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

const uint16_t* bf16(const at::Tensor& t) { return t.defined() ? (const uint16_t*)t.data_ptr() : nullptr; }

// Whether strided tensors share memory, exactly: is there a t with
// distance + sum_i step_i t_i = 0 and low_i <= t_i <= high_i? Steps are taken
// from the largest down; what the smaller ones can still add bounds each t_i to
// a few values where dimensions lie inside one another, as views' do. Layouts
// so entangled that the search is long count as sharing.
class Reach {
 public:
  void add(int64_t step, int64_t low, int64_t high) {
    if (low == high && low == 0) return;
    for (Term& t : terms_)
      if (t.step == step) {
        t.low += low, t.high += high;
        return;
      }
    terms_.push_back({step, low, high});
  }
  bool zero(int64_t distance) {
    std::sort(terms_.begin(), terms_.end(), [](const Term& a, const Term& b) { return a.step > b.step; });
    const size_t n = terms_.size();
    rest_low_.assign(n + 1, 0), rest_high_.assign(n + 1, 0);
    for (size_t i = n; i-- > 0;) {
      rest_low_[i] = rest_low_[i + 1] + terms_[i].step * terms_[i].low;
      rest_high_[i] = rest_high_[i + 1] + terms_[i].step * terms_[i].high;
    }
    left_ = 1 << 18;
    return from(0, distance);
  }

 private:
  struct Term {
    int64_t step, low, high;
  };
  static int64_t floor_div(int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
  bool from(size_t i, int64_t d) {
    if (i == terms_.size()) return d == 0;
    const Term& t = terms_[i];
    if (t.step == 0) return from(i + 1, d);
    const int64_t first = std::max(t.low, -floor_div(d + rest_high_[i + 1], t.step));
    const int64_t last = std::min(t.high, floor_div(-d - rest_low_[i + 1], t.step));
    for (int64_t v = first; v <= last; ++v) {
      if (--left_ < 0) return true;
      if (from(i + 1, d + v * t.step)) return true;
    }
    return false;
  }
  std::vector<Term> terms_;
  std::vector<int64_t> rest_low_, rest_high_;
  int64_t left_ = 0;
};

int64_t byte_stride(const at::Tensor& t, int64_t d) { return t.stride(d) * (int64_t)t.element_size(); }

// A tensor's bytes, from the first to behind the last: none of one that is undefined or empty.
struct Place {
  const at::Tensor* t;
  int64_t begin = 0, end = 0;
  explicit Place(const at::Tensor& tensor) : t(&tensor) {
    if (!t->defined() || t->numel() == 0) return;
    const at::IntArrayRef sizes = t->sizes(), strides = t->strides();
    int64_t last = 0;
    for (size_t d = 0; d < sizes.size(); ++d) last += (sizes[d] - 1) * strides[d];
    begin = (int64_t)reinterpret_cast<uintptr_t>(t->const_data_ptr());
    end = begin + (last + 1) * (int64_t)t->element_size();
  }
};

bool share_memory(const Place& pa, const Place& pb) {
  if (pa.end <= pb.begin || pb.end <= pa.begin) return false;
  const at::Tensor &a = *pa.t, &b = *pb.t;
  if (a.device() != b.device()) return false;
  Reach r;
  for (int64_t d = 0; d < a.dim(); ++d) r.add(byte_stride(a, d), -(a.size(d) - 1), 0);
  for (int64_t d = 0; d < b.dim(); ++d) r.add(byte_stride(b, d), 0, b.size(d) - 1);
  r.add(1, -((int64_t)a.element_size() - 1), (int64_t)b.element_size() - 1);
  return r.zero(pb.begin - pa.begin);
}

// Whether two places of a tensor are one: two index vectors that differ first
// in dimension `d` (by 1 and more; the others by anything) and meet.
bool shares_itself(const at::Tensor& t) {
  if (t.numel() < 2) return false;
  const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
  // Nearly all tensors' dimensions lie inside one another in their order: each
  // stride is beyond all that the ones behind it reach.
  int64_t reach = 0;
  bool nested = true;
  for (size_t d = sizes.size(); d-- > 0;) {
    if (sizes[d] < 2) continue;
    nested = nested && strides[d] > reach;
    reach += (sizes[d] - 1) * strides[d];
  }
  if (nested) return false;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (sizes[d] < 2) continue;
    if (strides[d] == 0) return true;
    Reach r;
    for (int64_t e = d + 1; e < t.dim(); ++e) r.add(byte_stride(t, e), -(t.size(e) - 1), t.size(e) - 1);
    r.add(byte_stride(t, d), 0, t.size(d) - 2);
    if (r.zero(byte_stride(t, d))) return true;
  }
  return false;
}

// What a call writes lies apart from what it reads and from what else it
// writes, and no two places of it are one.
struct Written {
  const at::Tensor* t;
  const char* name;
};
void check_written(std::initializer_list<Written> written, std::initializer_list<const at::Tensor*> read, const char* what) {
  c10::SmallVector<Place, 4> mine;
  for (const Written& w : written) {
    if (w.t->defined()) TORCH_CHECK(!shares_itself(*w.t), what, ": ", w.name, " must not overlap itself");
    mine.emplace_back(*w.t);
  }
  for (size_t i = 0; i < mine.size(); ++i)
    for (size_t j = 0; j < i; ++j)
      TORCH_CHECK(!share_memory(mine[i], mine[j]), what, ": ", written.begin()[i].name, " must not overlap ", written.begin()[j].name);
  for (const at::Tensor* t : read) {
    const Place p(*t);
    for (size_t i = 0; i < mine.size(); ++i)
      TORCH_CHECK(!share_memory(mine[i], p), what, ": ", written.begin()[i].name, " must not overlap the call's inputs");
  }
}

// A caller's output, or a new one. `direct` is what the kernel writes: the
// output itself where its rows can be stored in place, else a copy of it that
// is copied back (so that rows the call leaves alone keep their values).
struct Out {
  at::Tensor result, direct;
  bool given = false;
};
Out output(const OptTensor& out, at::IntArrayRef sizes, const at::Tensor& like, int64_t unit, const char* what) {
  Out o;
  if (!has(out)) {
    o.result = o.direct = at::empty(sizes, like.options());
    return o;
  }
  o.given = true;
  o.result = *out;
  o.direct = rows_ok(o.result, unit) ? o.result : o.result.contiguous().clone();
  return o;
}
void check_output(const OptTensor& out, at::IntArrayRef sizes, const char* what) {
  if (!has(out)) return;
  TORCH_CHECK_TYPE(out->scalar_type() == at::kBFloat16, what, ": out must be bfloat16, got ", out->scalar_type());
  TORCH_CHECK_VALUE(out->sizes() == sizes, what, ": out must be ", sizes, ", got ", out->sizes());
  TORCH_CHECK(!out->requires_grad() && !has_tangent(*out), what, ": out with requires_grad=True is not supported, nor one with a tangent");
}
void finish(Out& o) {
  if (!o.direct.is_same(o.result))
    o.result.copy_(o.direct);
  else if (o.given)
    was_written(o.result);
}

void check_table(const at::Tensor& cos_sin) {
  check_dtype(cos_sin, at::kFloat, "cos_sin");
  check_dim(cos_sin, 2, "cos_sin", "[positions, rope_dim]");
  TORCH_CHECK_VALUE(cos_sin.size(1) % 2 == 0, "cos_sin must have an even number of columns, got ", cos_sin.size(1));
}
// Rows of whole 16-byte pieces.
at::Tensor table_rows(const at::Tensor& cos_sin) { return rows_for(cos_sin.contiguous(), 4); }

void check_eps(double eps, const char* what) {
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, what, ": eps must be finite and not negative, got ", eps);
}
void check_scale(double scale, const char* what) {
  const float f = (float)scale;
  TORCH_CHECK_VALUE(std::isfinite(f) && f > 0, what, ": scale must be positive and finite, got ", scale);
}

at::Tensor head_norm_rope(at::Tensor x, at::Tensor positions, at::Tensor cos_sin, OptTensor weight, double eps,
                          bool normalize, bool inverse, bool interleaved, OptTensor out) {
  const char* what = "head_norm_rope";
  check_dtype(x, at::kBFloat16, "x");
  check_dim(x, 3, "x", "[tokens, heads, dim]");
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  TORCH_CHECK_VALUE(H > 0 && D > 0 && D <= 65536 && H <= 65536, "x must have 1 to 65536 heads of 1 to 65536 values, got ",
                    x.sizes());
  check_index(positions, T, "positions");
  check_table(cos_sin);
  TORCH_CHECK_VALUE(cos_sin.size(1) <= D, "cos_sin rotates ", cos_sin.size(1), " values of heads of ", D);
  check_eps(eps, what);
  if (has(weight)) {
    TORCH_CHECK_VALUE(normalize, "weight needs normalize=True");
    check_dtype(*weight, at::kBFloat16, "weight");
    TORCH_CHECK_VALUE(weight->dim() == 1 && weight->size(0) == D, "weight must be [", D, "], got ", weight->sizes());
  }
  check_output(out, x.sizes(), what);
  const at::Tensor w = opt(weight), given = opt(out);
  check_no_grad({&x, &cos_sin, &w}, what);
  // in place: a row is read by the lanes that write it, before they do
  const bool in_place = given.defined() && given.data_ptr() == x.data_ptr() && stride_at(given, 0) == stride_at(x, 0) &&
                        stride_at(given, 1) == stride_at(x, 1) && stride_at(given, 2) == stride_at(x, 2);
  const at::Tensor none;
  if (given.defined())
    check_written({{&given, "out (unless it is x itself)"}}, {in_place ? &none : &x, &positions, &cos_sin, &w}, what);
  check_devices(x, {&positions, &cos_sin, &w, &given}, what);
  c10::DeviceGuard guard(x.device());
  Out o = output(out, x.sizes(), x, 1, what);
  if (T == 0) return o.result;
  const at::Tensor xs = x.size(2) > 1 && x.stride(2) != 1 ? x.contiguous() : x;
  const at::Tensor pos = positions.contiguous(), table = table_rows(cos_sin);
  const at::Tensor ws = w.defined() ? rows_for(w.contiguous(), 8) : w;
  fcmoe_head_norm_rope_args a{};
  a.x = bf16(xs);
  a.tokens = T, a.heads = H, a.dim = D;
  a.x_token_stride = stride_at(xs, 0), a.x_head_stride = stride_at(xs, 1);
  a.positions = pos.data_ptr(), a.positions_i64 = pos.scalar_type() == at::kLong;
  a.cos_sin = table.size(1) ? table.data_ptr<float>() : nullptr;
  a.table_rows = table.size(0), a.rope_dim = table.size(1);
  a.weight = bf16(ws), a.eps = (float)eps;
  a.normalize = normalize, a.inverse = inverse, a.interleaved = interleaved;
  a.out = (uint16_t*)o.direct.data_ptr();
  a.out_token_stride = stride_at(o.direct, 0), a.out_head_stride = stride_at(o.direct, 1);
  {
    pybind11::gil_scoped_release release;
    check_rc(fcmoe_head_norm_rope(&a, stream_of(x)), what);
  }
  finish(o);
  return o.result;
}

// The cache's shapes; its device pointers once the devices are known to match.
fcmoe_latent_cache check_cache(const at::Tensor& latent, const at::Tensor& rope, const at::Tensor& scale,
                               const char* what) {
  TORCH_CHECK_TYPE(latent.scalar_type() == at::kBFloat16 || latent.scalar_type() == at::kFloat8_e4m3fn, what,
                   ": cache.latent must be bfloat16 or float8_e4m3fn, got ", latent.scalar_type());
  check_dim(latent, 3, "cache.latent", "[pages, page_size, latent_dim]");
  fcmoe_latent_cache c{};
  c.e4m3 = latent.scalar_type() == at::kFloat8_e4m3fn;
  c.pages = latent.size(0), c.page_size = latent.size(1), c.latent_dim = latent.size(2);
  TORCH_CHECK_VALUE(c.latent_dim == 256 || c.latent_dim == 512, "cache.latent_dim must be 256 or 512, got ", c.latent_dim);
  TORCH_CHECK_VALUE(c.page_size > 0 && c.page_size <= (1 << 20), "cache pages must hold 1 to 2^20 tokens, got ", c.page_size);
  const int64_t unit = c.e4m3 ? 16 : 8;
  TORCH_CHECK_VALUE(rows_ok(latent, unit), "cache.latent rows must be contiguous and start at multiples of 16 bytes");
  if (rope.defined()) {
    TORCH_CHECK_TYPE(rope.scalar_type() == latent.scalar_type(), "cache.rope must have cache.latent's dtype, got ",
                     rope.scalar_type());
    TORCH_CHECK_VALUE(rope.dim() == 3 && rope.size(0) == c.pages && rope.size(1) == c.page_size && rope.size(2) == 64,
                      "cache.rope must be [", c.pages, ", ", c.page_size, ", 64], got ", rope.sizes());
    TORCH_CHECK_VALUE(rows_ok(rope, unit), "cache.rope rows must be contiguous and start at multiples of 16 bytes");
    c.rope_dim = 64;
    c.rope_page_stride = stride_at(rope, 0), c.rope_row_stride = stride_at(rope, 1);
  }
  TORCH_CHECK_VALUE(scale.defined() == (c.e4m3 != 0), "cache.scale goes with a float8_e4m3fn cache and no other");
  if (scale.defined()) {
    check_dtype(scale, at::kFloat, "cache.scale");
    TORCH_CHECK_VALUE(scale.dim() == 2 && scale.size(0) == c.pages && scale.size(1) == c.page_size &&
                          (c.page_size == 1 || scale.stride(1) == 1),
                      "cache.scale must be [", c.pages, ", ", c.page_size, "] with contiguous pages, got ", scale.sizes());
    c.scale_page_stride = stride_at(scale, 0);
  }
  c.latent_page_stride = stride_at(latent, 0), c.latent_row_stride = stride_at(latent, 1);
  return c;
}
void cache_pointers(fcmoe_latent_cache& c, const at::Tensor& latent, const at::Tensor& rope, const at::Tensor& scale) {
  c.latent = latent.data_ptr();
  c.rope = rope.defined() ? rope.data_ptr() : nullptr;
  c.scale = scale.defined() ? scale.data_ptr<float>() : nullptr;
}

OptTensor latent_cache_append(at::Tensor kv, at::Tensor positions, at::Tensor slots, at::Tensor cos_sin,
                              at::Tensor latent, OptTensor rope_, OptTensor scale_, OptTensor weight, double eps,
                              bool interleaved, bool return_rows) {
  const char* what = "latent_cache_append";
  const at::Tensor rope = opt(rope_), scale = opt(scale_), w = opt(weight);
  fcmoe_latent_append_args a{};
  a.cache = check_cache(latent, rope, scale, what);
  check_dtype(kv, at::kBFloat16, "kv");
  const int64_t W = a.cache.latent_dim + a.cache.rope_dim;
  TORCH_CHECK_VALUE(kv.dim() == 2 && kv.size(1) == W, "kv must be [tokens, ", W, "], got ", kv.sizes());
  const int64_t T = kv.size(0);
  check_index(positions, T, "positions");
  check_index(slots, T, "slots");
  check_table(cos_sin);
  if (a.cache.rope_dim) {
    TORCH_CHECK_VALUE(cos_sin.size(1) == a.cache.rope_dim, "cos_sin must have rope_dim = ", a.cache.rope_dim,
                      " columns, got ", cos_sin.size(1));
  } else {
    TORCH_CHECK_VALUE(cos_sin.size(1) % 16 == 0 && cos_sin.size(1) <= a.cache.latent_dim,
                      "cos_sin must have a multiple of 16 columns, at most latent_dim = ", a.cache.latent_dim, ", got ",
                      cos_sin.size(1));
  }
  check_eps(eps, what);
  if (w.defined()) {
    check_dtype(w, at::kBFloat16, "weight");
    TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == a.cache.latent_dim, "weight must be [", a.cache.latent_dim, "], got ",
                      w.sizes());
  }
  check_no_grad({&kv, &cos_sin, &w, &latent, &rope, &scale}, what);
  check_written({{&latent, "cache.latent"}, {&rope, "cache.rope"}, {&scale, "cache.scale"}},
                {&kv, &positions, &slots, &cos_sin, &w}, what);
  check_devices(kv, {&positions, &slots, &cos_sin, &latent, &rope, &scale, &w}, what);
  c10::DeviceGuard guard(kv.device());
  OptTensor rows;
  if (return_rows) rows = at::empty({T, W}, kv.options());
  if (T == 0) return rows;
  cache_pointers(a.cache, latent, rope, scale);
  const at::Tensor in = rows_for(kv, 8), pos = positions.contiguous(), at_slots = slots.contiguous();
  const at::Tensor table = table_rows(cos_sin);
  const at::Tensor ws = w.defined() ? rows_for(w.contiguous(), 8) : w;
  a.kv = bf16(in), a.tokens = T, a.kv_row_stride = stride_at(in, 0);
  a.positions = pos.data_ptr(), a.slots = at_slots.data_ptr();
  a.positions_i64 = pos.scalar_type() == at::kLong, a.slots_i64 = at_slots.scalar_type() == at::kLong;
  a.cos_sin = table.size(1) ? table.data_ptr<float>() : nullptr;
  a.table_rows = table.size(0), a.rot_dim = table.size(1);
  a.weight = bf16(ws), a.eps = (float)eps, a.interleaved = interleaved;
  a.rows_out = return_rows ? (uint16_t*)rows->data_ptr() : nullptr;
  {
    pybind11::gil_scoped_release release;
    check_rc(fcmoe_latent_cache_append(&a, stream_of(kv)), what);
  }
  was_written(latent);
  was_written(rope);
  was_written(scale);
  return rows;
}

std::tuple<at::Tensor, int64_t, int64_t, int64_t> prepare_head_projection(at::Tensor weight) {
  const char* what = "prepare_head_projection";
  check_dtype(weight, at::kBFloat16, "weight");
  check_dim(weight, 3, "weight", "[heads, n, k]");
  const int64_t H = weight.size(0), N = weight.size(1), K = weight.size(2);
  TORCH_CHECK_VALUE(H > 0 && H <= 65535 && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0 && N <= 65536 && K <= 65536,
                    "weight must be [heads, n, k] with n and k multiples of 8, got ", weight.sizes());
  check_no_grad({&weight}, what);
  check_devices(weight, {}, what);
  c10::DeviceGuard guard(weight.device());
  const at::Tensor w = weight.contiguous();
  at::Tensor packed = at::empty({H, fcmoe_packed_expert_bytes(2, N, K, 1)}, w.options().dtype(at::kChar));
  check_rc(fcmoe_pack_experts(w.data_ptr(), 2, H, N, K, 1, packed.data_ptr(), stream_of(w)), what);
  return {packed, H, N, K};
}

at::Tensor head_projection(at::Tensor x, at::Tensor packed, int64_t heads, int64_t n, int64_t k, OptTensor out) {
  const char* what = "head_projection";
  check_dtype(x, at::kBFloat16, "x");
  TORCH_CHECK_VALUE(x.dim() == 3 && x.size(1) == heads && x.size(2) == k, "x must be [tokens, ", heads, ", ", k, "], got ",
                    x.sizes());
  const int64_t T = x.size(0);
  TORCH_CHECK_VALUE(packed.scalar_type() == at::kChar && packed.is_contiguous() &&
                        packed.numel() == heads * fcmoe_packed_expert_bytes(2, n, k, 1),
                    "weight must come from prepare_head_projection");
  check_output(out, {T, heads, n}, what);
  const at::Tensor given = opt(out);
  check_no_grad({&x}, what);
  if (given.defined()) check_written({{&given, "out"}}, {&x, &packed}, what);
  check_devices(x, {&packed, &given}, what);
  c10::DeviceGuard guard(x.device());
  Out o = output(out, {T, heads, n}, x, 4, what);
  if (T == 0) return o.result;
  const at::Tensor xs = rows_for(x, 8);
  fcmoe_head_projection_args a{};
  a.x = bf16(xs), a.tokens = T, a.heads = heads, a.n = n, a.k = k;
  a.x_token_stride = stride_at(xs, 0), a.x_head_stride = stride_at(xs, 1);
  a.w_packed = packed.data_ptr();
  a.out = (uint16_t*)o.direct.data_ptr();
  a.out_token_stride = stride_at(o.direct, 0), a.out_head_stride = stride_at(o.direct, 1);
  {
    pybind11::gil_scoped_release release;
    check_rc(fcmoe_head_projection(&a, stream_of(x)), what);
  }
  finish(o);
  return o.result;
}

// Tokens of a batch without sequences belong to none.
std::tuple<at::Tensor, OptTensor> no_sequences(Out& o, OptTensor lse) {
  if (!o.given) o.result.zero_();
  if (lse.has_value()) lse->fill_(-INFINITY);
  return {o.result, lse};
}

void check_starts(const at::Tensor& t, int64_t batch, const char* name) {
  check_dtype(t, at::kInt, name);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == batch + 1, name, " must be [", batch + 1, "], got ", t.sizes());
}

std::tuple<at::Tensor, OptTensor> absorbed_attention(at::Tensor q_latent, OptTensor q_rope_, at::Tensor latent,
                                                     OptTensor rope_, OptTensor scale_, at::Tensor page_table,
                                                     at::Tensor kv_lens, OptTensor query_starts, double scale,
                                                     OptTensor out, bool return_lse) {
  const char* what = "absorbed_attention";
  const at::Tensor q_rope = opt(q_rope_), rope = opt(rope_), cache_scale = opt(scale_), starts = opt(query_starts);
  fcmoe_absorbed_args a{};
  a.cache = check_cache(latent, rope, cache_scale, what);
  check_dtype(q_latent, at::kBFloat16, "q_latent");
  TORCH_CHECK_VALUE(q_latent.dim() == 3 && q_latent.size(1) > 0 && q_latent.size(1) <= 65536 &&
                        q_latent.size(2) == a.cache.latent_dim,
                    "q_latent must be [tokens, heads, ", a.cache.latent_dim, "], got ", q_latent.sizes());
  const int64_t T = q_latent.size(0), H = q_latent.size(1), R = q_latent.size(2);
  TORCH_CHECK_VALUE(q_rope.defined() == rope.defined(), "q_rope goes with a cache that has a rope part");
  if (q_rope.defined()) {
    check_dtype(q_rope, at::kBFloat16, "q_rope");
    TORCH_CHECK_VALUE(q_rope.dim() == 3 && q_rope.size(0) == T && q_rope.size(1) == H && q_rope.size(2) == a.cache.rope_dim,
                      "q_rope must be [", T, ", ", H, ", ", a.cache.rope_dim, "], got ", q_rope.sizes());
  }
  check_dtype(page_table, at::kInt, "page_table");
  check_dim(page_table, 2, "page_table", "[sequences, pages]");
  const int64_t B = page_table.size(0);
  check_dtype(kv_lens, at::kInt, "kv_lens");
  TORCH_CHECK_VALUE(kv_lens.dim() == 1 && kv_lens.size(0) == B, "kv_lens must be [", B, "], got ", kv_lens.sizes());
  if (starts.defined()) {
    check_starts(starts, B, "query_starts");
  } else {
    TORCH_CHECK_VALUE(T == B, "without query_starts there is one query token a sequence: got ", T, " and ", B);
  }
  TORCH_CHECK_VALUE(B <= (1 << 20) && T * H <= INT32_MAX / 2, "too many sequences or query rows");
  check_scale(scale, what);
  check_output(out, {T, H, R}, what);
  const at::Tensor given = opt(out);
  check_no_grad({&q_latent, &q_rope, &latent, &rope, &cache_scale}, what);
  if (given.defined())
    check_written({{&given, "out"}}, {&q_latent, &q_rope, &latent, &rope, &cache_scale, &page_table, &kv_lens, &starts},
                  what);
  check_devices(q_latent, {&q_rope, &latent, &rope, &cache_scale, &page_table, &kv_lens, &starts, &given}, what);
  c10::DeviceGuard guard(q_latent.device());
  Out o = output(out, {T, H, R}, q_latent, 4, what);
  OptTensor lse;
  if (return_lse) lse = at::empty({T, H}, q_latent.options().dtype(at::kFloat));
  if (T == 0) return {o.result, lse};
  if (B == 0) return no_sequences(o, lse);
  if (return_lse && o.given && starts.defined()) lse->fill_(-INFINITY);  // rows that `out` keeps have no sum
  cache_pointers(a.cache, latent, rope, cache_scale);
  const at::Tensor ql = rows_for(q_latent, 8), qr = q_rope.defined() ? rows_for(q_rope, 8) : q_rope;
  const at::Tensor table = page_table.size(1) > 1 && page_table.stride(1) != 1 ? page_table.contiguous() : page_table;
  const at::Tensor lens = kv_lens.contiguous(), st = starts.defined() ? starts.contiguous() : starts;
  a.q_latent = bf16(ql), a.q_rope = bf16(qr);
  a.tokens = T, a.heads = H, a.batch = B;
  a.q_latent_token_stride = stride_at(ql, 0), a.q_latent_head_stride = stride_at(ql, 1);
  if (qr.defined()) a.q_rope_token_stride = stride_at(qr, 0), a.q_rope_head_stride = stride_at(qr, 1);
  a.page_table = table.data_ptr<int32_t>(), a.table_width = table.size(1), a.page_table_stride = stride_at(table, 0);
  a.kv_lens = lens.data_ptr<int32_t>(), a.query_starts = st.defined() ? st.data_ptr<int32_t>() : nullptr;
  a.scale = (float)scale;
  a.out = (uint16_t*)o.direct.data_ptr();
  a.out_token_stride = stride_at(o.direct, 0), a.out_head_stride = stride_at(o.direct, 1);
  a.lse = return_lse ? lse->data_ptr<float>() : nullptr;
  a.zero_uncovered = !o.given;
  a.workspace_bytes = fcmoe_absorbed_attention_workspace_bytes(&a);
  at::Tensor ws = at::empty({(int64_t)a.workspace_bytes}, q_latent.options().dtype(at::kByte));
  a.workspace = ws.data_ptr();
  {
    pybind11::gil_scoped_release release;
    check_rc(fcmoe_absorbed_attention(&a, stream_of(q_latent)), what);
  }
  finish(o);
  return {o.result, lse};
}

std::tuple<at::Tensor, OptTensor> expanded_attention(at::Tensor q, at::Tensor kv, OptTensor k_rope_,
                                                     at::Tensor query_starts, OptTensor kv_starts_, double scale,
                                                     bool causal, OptTensor out, bool return_lse) {
  const char* what = "expanded_attention";
  const at::Tensor k_rope = opt(k_rope_);
  const at::Tensor kv_starts = has(kv_starts_) ? *kv_starts_ : query_starts;
  check_dtype(q, at::kBFloat16, "q");
  check_dtype(kv, at::kBFloat16, "kv");
  check_dim(q, 3, "q", "[tokens, heads, nope + rope_dim]");
  const int64_t T = q.size(0), H = q.size(1);
  TORCH_CHECK_VALUE(H > 0 && H <= 65536, "q must have 1 to 65536 heads, got ", q.sizes());
  TORCH_CHECK_VALUE(kv.dim() == 3 && kv.size(1) == H, "kv must be [keys, ", H, ", nope + v], got ", kv.sizes());
  const int64_t S = kv.size(0);
  int64_t P = 0;
  if (k_rope.defined()) {
    check_dtype(k_rope, at::kBFloat16, "k_rope");
    TORCH_CHECK_VALUE(k_rope.dim() == 2 && k_rope.size(0) == S && k_rope.size(1) == 64, "k_rope must be [", S,
                      ", 64], got ", k_rope.sizes());
    P = 64;
  }
  const int64_t N = q.size(2) - P, V = kv.size(2) - N;
  TORCH_CHECK_VALUE((N == 128 && V == 128) || (N == 64 && V == 64),
                    "head sizes (nope, v) must be (128, 128) or (64, 64), got (", N, ", ", V, ") from q ", q.sizes(), ", kv ",
                    kv.sizes(), " and rope_dim ", P);
  TORCH_CHECK_VALUE(T <= INT32_MAX && S <= INT32_MAX, "too many tokens");
  check_dtype(query_starts, at::kInt, "query_starts");
  TORCH_CHECK_VALUE(query_starts.dim() == 1 && query_starts.size(0) >= 1, "query_starts must be [sequences + 1], got ",
                    query_starts.sizes());
  const int64_t B = query_starts.size(0) - 1;
  TORCH_CHECK_VALUE(B <= (1 << 20), "too many sequences");
  check_starts(kv_starts, B, "kv_starts");
  check_scale(scale, what);
  check_output(out, {T, H, V}, what);
  const at::Tensor given = opt(out);
  check_no_grad({&q, &kv, &k_rope}, what);
  if (given.defined()) check_written({{&given, "out"}}, {&q, &kv, &k_rope, &query_starts, &kv_starts}, what);
  check_devices(q, {&kv, &k_rope, &query_starts, &kv_starts, &given}, what);
  c10::DeviceGuard guard(q.device());
  Out o = output(out, {T, H, V}, q, 4, what);
  OptTensor lse;
  if (return_lse) lse = at::empty({T, H}, q.options().dtype(at::kFloat));
  if (T == 0) return {o.result, lse};
  if (B == 0) return no_sequences(o, lse);
  if (return_lse && o.given) lse->fill_(-INFINITY);  // rows that `out` keeps have no sum
  const at::Tensor qs = rows_for(q, 8);
  // a tile's rows are addressed by 32-bit offsets from its first
  auto near = [](const at::Tensor& t) { return rows_ok(t, 8) && stride_at(t, 0) < (1 << 24) ? t : t.contiguous().clone(); };
  const at::Tensor kvs = near(kv), rs = k_rope.defined() ? near(k_rope) : k_rope;
  const at::Tensor st = query_starts.contiguous(), kst = kv_starts.contiguous();
  fcmoe_expanded_args a{};
  a.q = bf16(qs), a.kv = S ? bf16(kvs) : nullptr, a.k_rope = S && P ? bf16(rs) : nullptr;
  a.tokens = T, a.keys = S, a.heads = H, a.batch = B;
  a.nope_dim = N, a.rope_dim = P, a.v_dim = V;
  a.q_token_stride = stride_at(qs, 0), a.q_head_stride = stride_at(qs, 1);
  a.kv_token_stride = stride_at(kvs, 0), a.kv_head_stride = stride_at(kvs, 1);
  if (P) a.k_rope_token_stride = stride_at(rs, 0);
  a.query_starts = st.data_ptr<int32_t>(), a.kv_starts = kst.data_ptr<int32_t>();
  a.scale = (float)scale, a.causal = causal;
  a.out = (uint16_t*)o.direct.data_ptr();
  a.out_token_stride = stride_at(o.direct, 0), a.out_head_stride = stride_at(o.direct, 1);
  a.lse = return_lse ? lse->data_ptr<float>() : nullptr;
  a.zero_uncovered = !o.given;
  a.workspace_bytes = fcmoe_expanded_attention_workspace_bytes(&a);
  at::Tensor ws;
  if (a.workspace_bytes) {
    ws = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
  }
  {
    pybind11::gil_scoped_release release;
    check_rc(fcmoe_expanded_attention(&a, stream_of(q)), what);
  }
  finish(o);
  return {o.result, lse};
}

}  // namespace

void bind_latent_attention(pybind11::module_& m) {
  m.def("latent_head_norm_rope", &head_norm_rope);
  m.def("latent_cache_append", &latent_cache_append);
  m.def("latent_prepare_head_projection", &prepare_head_projection);
  m.def("latent_head_projection", &head_projection);
  m.def("latent_absorbed_attention", &absorbed_attention);
  m.def("latent_expanded_attention", &expanded_attention);
}
