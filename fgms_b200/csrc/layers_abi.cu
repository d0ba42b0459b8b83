// Entry points of what stands between and around layers of groups: norm, dropout, rows and products in 8 bits, a layer of experts for a few tokens
// (see include/fgms_b200.h for the contract of each).  They have no counterpart in the reference.
#include "../../include/fgms_b200.h"

#include <algorithm>
#include <cmath>

#include "host.cuh"
#include "dropout.cuh"
#include "expert_layer.cuh"
#include "grouped_i8.cuh"
#include "row_norm.cuh"

namespace fgms_host {
int take_layer_problems(int reset, unsigned long long* sum) { return take_problems(fgms::g_device_problems, reset, sum); }
}  // namespace fgms_host

namespace {

using namespace fgms_host;

bool layer_dtype_ok(int dtype) { return dtype == FGMS_DTYPE_F32 || dtype == FGMS_DTYPE_F16 || dtype == FGMS_DTYPE_BF16; }
size_t layer_elem(int dtype) { return dtype == FGMS_DTYPE_F32 ? 4 : 2; }

// Rows of `width` values in memory, `pitch` values apart (of a single row: whatever the caller says).
struct RowSpan {
  const void* p;
  int64_t rows, pitch, width;
  size_t es;
  RowSpan(const void* p_, int64_t rows_, int64_t pitch_, int64_t width_, size_t es_) : p(p_), rows(rows_), pitch(rows_ > 1 ? pitch_ : width_), width(width_), es(es_) {}
  bool any() const { return p != nullptr && rows > 0; }
  size_t bytes() const { return rows > 0 ? ((size_t)(rows - 1) * (size_t)pitch + (size_t)width) * es : 0; }
  // whether any value of one is a value of the other, except where both are the very same rows
  bool collides(const RowSpan& o) const {
    if (!any() || !o.any()) return false;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
    const size_t row = (size_t)pitch * es, mine = (size_t)width * es, its = (size_t)o.width * o.es;
    if (row == (size_t)o.pitch * o.es) {
      if (a == b && es == o.es && width == o.width) return false;
      const size_t apart = b > a ? (size_t)(b - a) % row : (row - (size_t)(a - b) % row) % row;  // columns side by side in the same rows
      if (apart >= mine && row - apart >= its) return false;
    }
    return Range{p, bytes()}.overlaps(Range{o.p, o.bytes()});
  }
  bool same(const RowSpan& o) const { return any() && o.any() && p == o.p; }
  bool on_boundary() const { return (reinterpret_cast<uintptr_t>(p) & (es - 1)) == 0; }
  bool vec(size_t boundary) const { return (reinterpret_cast<uintptr_t>(p) & (boundary - 1)) == 0 && (rows <= 1 || (size_t)pitch * es % boundary == 0); }
};

int check_span(const char* name, const RowSpan& s, bool needed) {
  if (!s.p) return needed && s.rows > 0 ? fail(FGMS_ERR_INVALID_ARG, "%s: null pointer", name) : FGMS_OK;
  if (s.rows > 1 && s.pitch < s.width) return fail(FGMS_ERR_INVALID_ARG, "%s: rows are %lld values apart, %lld wide", name, (long long)s.pitch, (long long)s.width);
  if (s.pitch > 0x7fffffffll * 16) return fail(FGMS_ERR_INVALID_ARG, "%s: rows too far apart", name);
  if (!s.on_boundary()) return fail(FGMS_ERR_INVALID_ARG, "%s is not on a boundary of its type", name);
  return FGMS_OK;
}

int check_rows(int64_t rows, int64_t width, int64_t most) {
  if (rows < 0 || rows > 0x7fffffffll) return fail(FGMS_ERR_INVALID_ARG, "rows %lld outside [0, 2^31 - 1]", (long long)rows);
  if (width < 1 || width > most) return fail(FGMS_ERR_INVALID_ARG, "width %lld outside [1, %lld]", (long long)width, (long long)most);
  return FGMS_OK;
}

// the lots below which a value is dropped
int drop_threshold(double p, uint32_t* threshold, float* factor) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(FGMS_ERR_INVALID_ARG, "the probability of dropping must be in [0, 1], got %g", p);
  *threshold = (uint32_t)std::lrint(p * 65536.0);
  *factor = *threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)*threshold)) : 0.f;
  return FGMS_OK;
}

int check_state(const char* name, const void* at, bool needed) {
  if (needed && !at) return fail(FGMS_ERR_INVALID_ARG, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(at) & 7) return fail(FGMS_ERR_INVALID_ARG, "%s is not on a boundary of its type", name);
  return FGMS_OK;
}

int run_dropout(const fgms_b200_dropout_args& a, bool backward, cudaStream_t st) {
  if (int rc = check_rows(a.rows, a.width, 0x7ffffff0ll)) return rc;
  if (!layer_dtype_ok(a.dtype)) return fail(FGMS_ERR_INVALID_ARG, "unknown dtype %d", a.dtype);
  fgms::DropoutParams p{};
  if (int rc = drop_threshold(a.p, &p.drop.threshold, &p.drop.factor)) return rc;
  const size_t es = layer_elem(a.dtype);
  const RowSpan x{a.x, a.rows, a.x_pitch, a.width, es}, residual{backward ? nullptr : a.residual, a.rows, a.residual_pitch, a.width, es},
      out{a.out, a.rows, a.out_pitch, a.width, es};
  if (int rc = check_span("x", x, true)) return rc;
  if (int rc = check_span("residual", residual, false)) return rc;
  if (int rc = check_span("out", out, true)) return rc;
  if (int rc = check_state("rng", a.rng, !backward)) return rc;
  if (int rc = check_state("rng_used", a.rng_used, backward)) return rc;
  if (out.collides(x) || out.collides(residual)) return fail(FGMS_ERR_INVALID_ARG, "the output overlaps an input");
  const Range written{a.out, out.bytes()}, state{a.rng, backward ? 0u : 24u}, used{a.rng_used, a.rng_used ? 16u : 0u};
  for (const Range& r : {state, used})
    if (r.p && r.bytes && (r.overlaps(written) || r.overlaps(Range{a.x, x.bytes()}) || (residual.any() && r.overlaps(Range{a.residual, residual.bytes()}))))
      return fail(FGMS_ERR_INVALID_ARG, "the generator's state overlaps a tensor");
  if (!backward && a.rng_used && state.overlaps(used)) return fail(FGMS_ERR_INVALID_ARG, "rng_used overlaps rng");
  if (a.rows == 0) return FGMS_OK;
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  p.x = a.x;
  p.residual = residual.p;
  p.out = a.out;
  p.rows = a.rows;
  p.width = (int)a.width;
  p.x_pitch = a.x_pitch;
  p.residual_pitch = a.residual_pitch;
  p.out_pitch = a.out_pitch;
  p.x_vec = x.vec(16);
  p.residual_vec = residual.vec(16);
  p.out_vec = out.vec(16);
  p.drop.state = reinterpret_cast<long long*>(a.rng);
  p.drop.used = reinterpret_cast<long long*>(a.rng_used);
  p.alone = di.reserved > 0;
  const long long chunks = a.rows * ((a.width + fgms::ROW_CHUNK - 1) / fgms::ROW_CHUNK);
  const long long blocks = (chunks + fgms::DROP_THREADS - 1) / fgms::DROP_THREADS, most = (long long)fgms::DROP_BLOCKS * di.sms;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  const auto launch = [&](auto type) {
    using T = decltype(type);
    const bool some = p.drop.threshold > 0;
    if (backward)
      return some ? fgms::launch_pdl(fgms::dropout_kernel<T, true, true>, grid, fgms::DROP_THREADS, 0, st, p)
                  : fgms::launch_pdl(fgms::dropout_kernel<T, true, false>, grid, fgms::DROP_THREADS, 0, st, p);
    return some ? fgms::launch_pdl(fgms::dropout_kernel<T, false, true>, grid, fgms::DROP_THREADS, 0, st, p)
                : fgms::launch_pdl(fgms::dropout_kernel<T, false, false>, grid, fgms::DROP_THREADS, 0, st, p);
  };
  const cudaError_t e = a.dtype == FGMS_DTYPE_F32 ? launch(float()) : a.dtype == FGMS_DTYPE_F16 ? launch(__half()) : launch(__nv_bfloat16());
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "dropout_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("dropout_kernel");
}

// the types of rows and weight that a norm is built for: the weight's is the rows' or fp32
template <typename F>
cudaError_t with_types(int dtype, int weight_dtype, F&& f) {
  if (dtype == FGMS_DTYPE_F32) return f(float(), float());
  if (dtype == FGMS_DTYPE_F16) return weight_dtype == FGMS_DTYPE_F32 ? f(__half(), float()) : f(__half(), __half());
  return weight_dtype == FGMS_DTYPE_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
}
int check_norm_types(int dtype, int weight_dtype) {
  if (!layer_dtype_ok(dtype)) return fail(FGMS_ERR_INVALID_ARG, "unknown dtype %d", dtype);
  if (weight_dtype != dtype && weight_dtype != FGMS_DTYPE_F32) return fail(FGMS_ERR_UNSUPPORTED, "the weight's type must be that of the rows, or fp32");
  return FGMS_OK;
}

int run_rms_norm(const fgms_b200_rms_norm_args& a, bool norm, cudaStream_t st) {
  if (int rc = check_rows(a.rows, a.width, fgms::NORM_MAX_WIDTH)) return rc;
  if (int rc = check_norm_types(a.dtype, norm ? a.weight_dtype : a.dtype)) return rc;
  if (norm && !(a.eps >= 0.0 && a.eps < 1e30)) return fail(FGMS_ERR_INVALID_ARG, "eps must be finite and not negative, got %g", a.eps);
  fgms::NormParams p{};
  if (int rc = drop_threshold(a.p, &p.drop.threshold, &p.drop.factor)) return rc;
  const bool eight = a.scale != nullptr, drop = p.drop.threshold > 0;
  if (eight && drop) return fail(FGMS_ERR_UNSUPPORTED, "no dropout with an output in 8 bits");
  const size_t es = layer_elem(a.dtype);
  const RowSpan x{a.x, a.rows, a.x_pitch, a.width, es}, residual{a.residual, a.rows, a.residual_pitch, a.width, es},
      out{a.out, a.rows, a.out_pitch, a.width, eight ? 1u : es}, sum{a.sum, a.rows, a.sum_pitch, a.width, es};
  const RowSpan weight{a.weight, 1, a.width, a.width, layer_elem(a.weight_dtype)}, scale{a.scale, 1, a.rows, a.rows, 4}, rstd{a.rstd, 1, a.rows, a.rows, 4};
  if (int rc = check_span("x", x, true)) return rc;
  if (int rc = check_span("residual", residual, false)) return rc;
  if (int rc = check_span("out", out, true)) return rc;
  if (int rc = check_span("sum", sum, false)) return rc;
  if (norm)
    if (int rc = check_span("weight", weight, true)) return rc;
  if (int rc = check_span("scale", scale, false)) return rc;
  if (int rc = check_span("rstd", rstd, false)) return rc;
  if (int rc = check_state("rng", a.rng, drop)) return rc;
  if (int rc = check_state("rng_used", a.rng_used, false)) return rc;
  if (a.rows == 0) return FGMS_OK;
  const RowSpan state{drop ? a.rng : nullptr, 1, 3, 3, 8}, used{drop ? a.rng_used : nullptr, 1, 2, 2, 8};
  const RowSpan outputs[] = {out, sum, scale, rstd, state, used}, inputs[] = {x, residual, weight};
  for (int i = 0; i < 6; ++i) {
    for (const RowSpan& in : inputs)
      if (outputs[i].collides(in) || (outputs[i].same(in) && (i >= 2 || &in == &inputs[2]))) return fail(FGMS_ERR_INVALID_ARG, "an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (outputs[i].collides(outputs[j]) || outputs[i].same(outputs[j])) return fail(FGMS_ERR_INVALID_ARG, "two outputs overlap");
  }
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  p.x = a.x;
  p.residual = a.residual;
  p.weight = a.weight;
  p.out = a.out;
  p.sum = a.sum;
  p.scale = a.scale;
  p.rstd = a.rstd;
  p.rows = a.rows;
  p.x_pitch = a.x_pitch;
  p.residual_pitch = a.residual_pitch;
  p.out_pitch = a.out_pitch;
  p.sum_pitch = a.sum_pitch;
  p.width = (int)a.width;
  p.norm = norm;
  p.x_vec = x.vec(16);
  p.residual_vec = residual.vec(16);
  p.out_vec = out.vec(eight ? 8 : 16);
  p.sum_vec = sum.vec(16);
  p.weight_vec = weight.vec(16);
  p.eps = (float)a.eps;
  p.inverse_width = 1.f / (float)a.width;
  p.drop.state = reinterpret_cast<long long*>(a.rng);
  p.drop.used = reinterpret_cast<long long*>(a.rng_used);
  p.alone = di.reserved > 0;
  const cudaError_t e = with_types(a.dtype, norm ? a.weight_dtype : a.dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    return eight ? fgms::launch_rms_norm<T, W, true>(p, st, di.sms) : fgms::launch_rms_norm<T, W, false>(p, st, di.sms);
  });
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "rms_norm_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("rms_norm_kernel");
}

int run_rms_norm_bwd(const fgms_b200_rms_norm_bwd_args& a, cudaStream_t st) {
  if (int rc = check_rows(a.rows, a.width, fgms::NORM_MAX_WIDTH)) return rc;
  if (int rc = check_norm_types(a.dtype, a.weight_dtype)) return rc;
  fgms::NormGradParams p{};
  if (int rc = drop_threshold(a.p, &p.drop.threshold, &p.drop.factor)) return rc;
  const bool drop = p.drop.threshold > 0;
  const size_t es = layer_elem(a.dtype);
  const auto span = [&](const void* at, int64_t pitch) { return RowSpan{at, a.rows, pitch, a.width, es}; };
  if (a.x && (a.dtype == FGMS_DTYPE_F32 || (a.weight_dtype != FGMS_DTYPE_F32 && a.sum)))
    return fail(FGMS_ERR_UNSUPPORTED, "x is read for rows in 16 bits, with a weight of their type where there is no sum; otherwise sum is");
  const RowSpan dy = span(a.out_grad, a.out_grad_pitch), h = a.x ? span(a.x, a.x_pitch) : span(a.sum, a.sum_pitch),
                residual = span(a.x ? a.residual : nullptr, a.residual_pitch), dsum = span(a.sum_grad, a.sum_grad_pitch), dx = span(a.x_grad, a.x_grad_pitch),
                dresidual = span(a.residual_grad, a.residual_grad_pitch);
  const RowSpan weight{a.weight, 1, a.width, a.width, layer_elem(a.weight_dtype)}, dw{a.weight_grad, 1, a.width, a.width, layer_elem(a.weight_dtype)},
      rstd{a.rstd, 1, a.rows, a.rows, 4};
  if (int rc = check_span("out_grad", dy, true)) return rc;
  if (int rc = check_span(a.x ? "x" : "sum", h, true)) return rc;
  if (int rc = check_span("residual", residual, false)) return rc;
  if (int rc = check_span("sum_grad", dsum, false)) return rc;
  if (int rc = check_span("x_grad", dx, false)) return rc;
  if (int rc = check_span("residual_grad", dresidual, false)) return rc;
  if (int rc = check_span("weight", weight, true)) return rc;
  if (int rc = check_span("weight_grad", dw, false)) return rc;
  if (int rc = check_span("rstd", rstd, a.rows > 0)) return rc;
  if (int rc = check_state("rng_used", a.rng_used, drop)) return rc;
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  const fgms::NormGradCut cut = fgms::norm_grad_cut(a.rows, (int)a.width, di.sms);
  const size_t needed = a.weight_grad ? (size_t)cut.blocks * (size_t)a.width * 4 : 0;
  if (needed > 0 && (!a.workspace || a.workspace_bytes < needed || (reinterpret_cast<uintptr_t>(a.workspace) & 15)))
    return fail(FGMS_ERR_WORKSPACE, "a workspace of %zu bytes on a 16-byte boundary is needed", needed);
  const RowSpan space{needed ? a.workspace : nullptr, 1, (int64_t)needed, (int64_t)needed, 1}, used{drop ? a.rng_used : nullptr, 1, 2, 2, 8};
  const RowSpan outputs[] = {dx, dresidual, dw, space}, inputs[] = {dy, h, dsum, residual, weight, rstd, used};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 7; ++j)
      if (outputs[i].collides(inputs[j]) || (outputs[i].same(inputs[j]) && (i >= 2 || j >= 4))) return fail(FGMS_ERR_INVALID_ARG, "an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (outputs[i].collides(outputs[j]) || outputs[i].same(outputs[j])) return fail(FGMS_ERR_INVALID_ARG, "two outputs overlap");
  }
  if (a.rows == 0) {  // no row adds anything to the weight's gradient
    if (a.weight_grad && cudaMemsetAsync(a.weight_grad, 0, dw.bytes(), st) != cudaSuccess)
      return fail(FGMS_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(cudaGetLastError()));
    return FGMS_OK;
  }
  p.dy = a.out_grad;
  p.sum = a.sum;
  p.x = a.x;
  p.residual = residual.p;
  p.dsum = a.sum_grad;
  p.weight = a.weight;
  p.rstd = a.rstd;
  p.dx = a.x_grad;
  p.dresidual = a.residual_grad;
  p.parts = a.weight_grad ? static_cast<float*>(a.workspace) : nullptr;
  p.rows = a.rows;
  p.dy_pitch = a.out_grad_pitch;
  p.sum_pitch = a.x ? a.x_pitch : a.sum_pitch;
  p.residual_pitch = a.residual_pitch;
  p.residual_vec = residual.vec(16);
  p.dsum_pitch = a.sum_grad_pitch;
  p.dx_pitch = a.x_grad_pitch;
  p.dresidual_pitch = a.residual_grad_pitch;
  p.width = (int)a.width;
  p.dy_vec = dy.vec(16);
  p.sum_vec = h.vec(16);
  p.dsum_vec = dsum.vec(16);
  p.dx_vec = dx.vec(16);
  p.dresidual_vec = dresidual.vec(16);
  p.weight_vec = weight.vec(16);
  p.inverse_width = 1.f / (float)a.width;
  p.drop.used = const_cast<long long*>(reinterpret_cast<const long long*>(a.rng_used));
  p.alone = di.reserved > 0;
  cudaError_t e = with_types(a.dtype, a.weight_dtype, [&](auto t, auto w) { return fgms::launch_rms_norm_grad<decltype(t), decltype(w)>(p, cut, st); });
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "rms_norm_grad_kernel: %s", cudaGetErrorString(e));
  }
  if (int rc = check_launch("rms_norm_grad_kernel")) return rc;
  if (!a.weight_grad) return FGMS_OK;
  const float* parts = p.parts;
  e = a.weight_dtype == FGMS_DTYPE_F32   ? fgms::launch_rms_norm_weight_grad<float>(parts, cut.blocks, p.width, a.weight_grad, p.alone, st)
      : a.weight_dtype == FGMS_DTYPE_F16 ? fgms::launch_rms_norm_weight_grad<__half>(parts, cut.blocks, p.width, a.weight_grad, p.alone, st)
                                         : fgms::launch_rms_norm_weight_grad<__nv_bfloat16>(parts, cut.blocks, p.width, a.weight_grad, p.alone, st);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "rms_norm_weight_grad_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("rms_norm_weight_grad_kernel");
}
// What of a product in 8 bits has to be copied to rows that a tensor map describes, and where to.
struct I8Copies {
  long long a_pitch, b_pitch;  // of the copies; 0: none is needed
  size_t a_at, b_at, total;
};
I8Copies i8_copies(const RowSpan& a, const RowSpan& b) {
  I8Copies c = {};
  const auto one = [&](const RowSpan& s, long long* pitch, size_t* at) {
    if (s.vec(16)) return;
    *pitch = (s.width + 15) / 16 * 16;
    *at = c.total;
    c.total += ((size_t)s.rows * (size_t)*pitch + 255) / 256 * 256;
  };
  one(a, &c.a_pitch, &c.a_at);
  one(b, &c.b_pitch, &c.b_at);
  return c;
}

int run_grouped_i8(const int8_t* codes, int64_t codes_pitch, const float* code_scale, const int8_t* kernel, int64_t kernel_pitch, const float* kernel_scale,
                   void* out, const int32_t* kpos, int n_rows, int c_in, int c_out, int groups, int dtype, int zero_rest, void* workspace,
                   size_t workspace_bytes, cudaStream_t st) {
  if (n_rows < 0) return fail(FGMS_ERR_INVALID_ARG, "negative row count");
  if (c_in < 1 || c_out < 1) return fail(FGMS_ERR_INVALID_ARG, "channel counts must be >= 1");
  if (c_in > fgms::GI_MAX_CONTRACTION) return fail(FGMS_ERR_INVALID_ARG, "more than %d channels to add up: their sum may leave an int32", fgms::GI_MAX_CONTRACTION);
  if (n_rows > FGMS_GROUPED_MAX_EXTENT || c_out > FGMS_GROUPED_MAX_EXTENT) return fail(FGMS_ERR_INVALID_ARG, "more than %d rows or channels", FGMS_GROUPED_MAX_EXTENT);
  if (groups < 1 || groups > FGMS_GROUPED_MAX_GROUPS) return fail(FGMS_ERR_INVALID_ARG, "groups %d outside [1, %d]", groups, FGMS_GROUPED_MAX_GROUPS);
  if ((long long)groups * c_out > 0x7fffffffll) return fail(FGMS_ERR_INVALID_ARG, "groups times channels exceeds the int32 range");
  if (((long long)n_rows / 64 + groups) * ((long long)c_out / 128 + 1) >= 0x7fff0000ll) return fail(FGMS_ERR_INVALID_ARG, "more tiles than an int32 counts");
  if (!layer_dtype_ok(dtype)) return fail(FGMS_ERR_INVALID_ARG, "unknown dtype %d", dtype);
  if (!kpos && groups != 1) return fail(FGMS_ERR_INVALID_ARG, "kpos may be null for a single group only");
  const size_t es = layer_elem(dtype);
  const RowSpan a{codes, n_rows, codes_pitch, c_in, 1}, b{kernel, (int64_t)groups * c_out, kernel_pitch, c_in, 1}, d{out, n_rows, c_out, c_out, es};
  const RowSpan sa{code_scale, 1, n_rows, n_rows, 4}, sb{kernel_scale, 1, (int64_t)groups * c_out, (int64_t)groups * c_out, 4}, k{kpos, 1, groups + 1, groups + 1, 4};
  if (int rc = check_span("codes", a, true)) return rc;
  if (int rc = check_span("kernel", b, true)) return rc;
  if (int rc = check_span("out", d, true)) return rc;
  if (int rc = check_span("code_scale", sa, n_rows > 0)) return rc;
  if (int rc = check_span("kernel_scale", sb, true)) return rc;
  if (int rc = check_span("kpos", k, false)) return rc;
  for (const RowSpan* in : {&a, &b, &sa, &sb, &k})
    if (d.collides(*in) || d.same(*in)) return fail(FGMS_ERR_INVALID_ARG, "the output overlaps an input");
  if (n_rows == 0) return FGMS_OK;
  const I8Copies copies = i8_copies(a, b);
  if (copies.total > 0) {
    if (!workspace || workspace_bytes < copies.total || (reinterpret_cast<uintptr_t>(workspace) & 255))
      return fail(FGMS_ERR_WORKSPACE, "rows that do not start on 16-byte boundaries need a workspace of %zu bytes on a 256-byte boundary", copies.total);
    const Range w{workspace, copies.total};
    for (const RowSpan* s : {&a, &b, &d, &sa, &sb, &k})
      if (s->any() && w.overlaps(Range{s->p, s->bytes()})) return fail(FGMS_ERR_WORKSPACE, "the workspace overlaps a tensor");
  }
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  fgms::GroupedI8Params q{};
  q.g.a = codes;
  q.g.b = kernel;
  q.g.d = out;
  q.g.kpos = kpos;
  q.g.n_rows = n_rows;
  q.g.c_in = c_out;
  q.g.c_out = (c_in + 1) / 2;
  q.g.groups = groups;
  q.g.zero_rest = zero_rest;
  q.g.d_pitch = c_out;
  q.g.alone = di.reserved > 0;
  q.row_scale = code_scale;
  q.channel_scale = kernel_scale;
  q.dtype = dtype == FGMS_DTYPE_F32 ? 0 : dtype == FGMS_DTYPE_F16 ? 1 : 2;
  q.store = !d.vec(16) ? 2 : dtype == FGMS_DTYPE_F32 ? 1 : 0;  // (contiguous rows: all of them on 16-byte boundaries, or a single one)
  if (c_out % (dtype == FGMS_DTYPE_F32 ? 4 : 8) != 0) q.store = 2;
  long long a_pitch = a.rows > 1 ? a.pitch : (c_in + 15) / 16 * 16, b_pitch = b.rows > 1 ? b.pitch : (c_in + 15) / 16 * 16;
  if (copies.total > 0) {
    uint8_t* to = static_cast<uint8_t*>(workspace);
    fgms::ByteRows x{}, y{};
    if (copies.a_pitch) {
      x = {reinterpret_cast<const uint8_t*>(codes), to + copies.a_at, a.rows, a.pitch, copies.a_pitch, c_in};
      q.g.a = x.dst;
      a_pitch = copies.a_pitch;
    }
    if (copies.b_pitch) {
      y = {reinterpret_cast<const uint8_t*>(kernel), to + copies.b_at, b.rows, b.pitch, copies.b_pitch, c_in};
      q.g.b = y.dst;
      b_pitch = copies.b_pitch;
    }
    const long long blocks = (x.rows + y.rows + 7) / 8, most = 8ll * di.sms;
    if (fgms::launch_pdl(fgms::copy_byte_rows_kernel, dim3((unsigned)(blocks < most ? blocks : most)), fgms::BR_THREADS, 0, st, x, y, q.g.alone) != cudaSuccess)
      return fail(FGMS_ERR_CUDA, "copy_byte_rows_kernel: %s", cudaGetErrorString(cudaGetLastError()));
    if (int rc = check_launch("copy_byte_rows_kernel")) return rc;
  }
  const int rc = fgms::launch_grouped_i8(q, c_in, a_pitch, b_pitch, st, di.sms, di.max_smem_optin);
  if (rc != 0) {
    const cudaError_t e = cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "grouped_i8_kernel: %s (%d)", cudaGetErrorString(e), rc);
  }
  return check_launch("grouped_i8_kernel");
}
int run_expert_layer(const fgms_b200_expert_layer_args& a, cudaStream_t st) {
  if (a.tokens < 0 || a.tokens > fgms::EL_MAX_TOKENS) return fail(FGMS_ERR_INVALID_ARG, "tokens %d outside [0, %d]", a.tokens, fgms::EL_MAX_TOKENS);
  if (a.experts < 1 || a.experts > fgms::EL_MAX_EXPERTS) return fail(FGMS_ERR_INVALID_ARG, "experts %d outside [1, %d]", a.experts, fgms::EL_MAX_EXPERTS);
  if (a.top_k < 1 || a.top_k > fgms::EL_MAX_TOP_K || a.top_k > a.experts)
    return fail(FGMS_ERR_INVALID_ARG, "top_k %d outside [1, %d], or more than the %d experts", a.top_k, fgms::EL_MAX_TOP_K, a.experts);
  for (const int c : {a.width, a.hidden, a.out_width})
    if (c < 8 || c > (1 << 20) || c % 8 != 0) return fail(FGMS_ERR_INVALID_ARG, "widths must be multiples of 8 up to 2^20, got %d", c);
  if (a.dtype != FGMS_DTYPE_F16 && a.dtype != FGMS_DTYPE_BF16) return fail(FGMS_ERR_UNSUPPORTED, "a layer of experts for a few tokens takes F16 or BF16");
  if (a.router_dtype != a.dtype && a.router_dtype != FGMS_DTYPE_F32) return fail(FGMS_ERR_UNSUPPORTED, "the router's type must be that of the rows, or fp32");
  if (a.activation != FGMS_ACTIVATION_RELU && a.activation != FGMS_ACTIVATION_SILU) return fail(FGMS_ERR_INVALID_ARG, "unknown activation %d", a.activation);
  const int64_t wide = a.gated ? 2ll * a.hidden : a.hidden;
  // (a tensor map's matrices are less than 2^40 bytes apart; items are then far from leaving an int)
  if ((int64_t)a.width * wide * 2 >= (1ll << 40) || (int64_t)a.hidden * a.out_width * 2 >= (1ll << 40)) return fail(FGMS_ERR_INVALID_ARG, "weights too large");
  const int64_t pairs = (int64_t)a.tokens * a.top_k;
  const RowSpan x{a.x, a.tokens, a.x_pitch, a.width, 2}, out{a.out, a.tokens, a.out_pitch, a.out_width, 2};
  const RowSpan router{a.router, a.experts, a.width, a.width, layer_elem(a.router_dtype)}, w_in{a.w_in, (int64_t)a.experts * a.width, wide, wide, 2},
      w_out{a.w_out, (int64_t)a.experts * a.hidden, a.out_width, a.out_width, 2};
  const RowSpan experts{a.chosen, 1, pairs, pairs, 4}, gates{a.gates, 1, pairs, pairs, 4};
  if (int rc = check_span("x", x, true)) return rc;
  if (int rc = check_span("router", router, true)) return rc;
  if (int rc = check_span("w_in", w_in, true)) return rc;
  if (int rc = check_span("w_out", w_out, true)) return rc;
  if (int rc = check_span("out", out, true)) return rc;
  if (int rc = check_span("chosen", experts, pairs > 0)) return rc;
  if (int rc = check_span("gates", gates, pairs > 0)) return rc;
  if (!x.vec(16) || !router.vec(16) || !w_in.vec(16) || !w_out.vec(16)) return fail(FGMS_ERR_INVALID_ARG, "rows and weights must start on 16-byte boundaries");
  if (a.tokens == 0) return FGMS_OK;
  const RowSpan outputs[] = {out, experts, gates}, inputs[] = {x, router, w_in, w_out};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < 4; ++j)
      if (outputs[i].collides(inputs[j]) || (outputs[i].same(inputs[j]) && (i > 0 || j > 0))) return fail(FGMS_ERR_INVALID_ARG, "an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (outputs[i].collides(outputs[j]) || outputs[i].same(outputs[j])) return fail(FGMS_ERR_INVALID_ARG, "two outputs overlap");
  }
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  const fgms::ExpertSpace space = fgms::expert_space(a.tokens, a.experts, a.top_k, a.hidden, a.out_width);
  if (!a.workspace || a.workspace_bytes < space.total || (reinterpret_cast<uintptr_t>(a.workspace) & 255))
    return fail(FGMS_ERR_WORKSPACE, "a workspace of %zu bytes on a 256-byte boundary is needed", space.total);
  for (const RowSpan* s : {&x, &router, &w_in, &w_out, &out, &experts, &gates})
    if (Range{a.workspace, space.total}.overlaps(Range{s->p, s->bytes()})) return fail(FGMS_ERR_WORKSPACE, "the workspace overlaps a tensor");
  uint8_t* at = static_cast<uint8_t*>(a.workspace);
  fgms::ExpertParams p{};
  p.x = a.x;
  p.router = a.router;
  p.out = a.out;
  p.experts = a.chosen;
  p.gates = a.gates;
  p.tokens = a.tokens;
  p.n_experts = a.experts;
  p.top_k = a.top_k;
  p.width = a.width;
  p.hidden = a.hidden;
  p.out_width = a.out_width;
  p.gated = a.gated != 0;
  p.activation = a.activation == FGMS_ACTIVATION_SILU;
  p.x_pitch = a.tokens > 1 ? a.x_pitch : a.width;
  p.out_pitch = a.tokens > 1 ? a.out_pitch : a.out_width;
  p.flags = reinterpret_cast<uint32_t*>(at + space.flags);
  p.h = reinterpret_cast<uint16_t*>(at + space.h);
  p.part = reinterpret_cast<float*>(at + space.part);
  p.ctas = di.sms;
  p.n_flags = space.n_flags;
  p.alone = di.reserved > 0;
  const cudaError_t e = with_types(a.dtype, a.router_dtype, [&](auto t, auto r) { return fgms::launch_expert_choice<decltype(t), decltype(r)>(p, st); });
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FGMS_ERR_CUDA, "expert_choice_kernel: %s", cudaGetErrorString(e));
  }
  if (int rc = check_launch("expert_choice_kernel")) return rc;
  const int rc = a.dtype == FGMS_DTYPE_BF16 ? fgms::launch_expert_layer<true>(p, a.w_in, a.w_out, st, di.max_smem_optin)
                                            : fgms::launch_expert_layer<false>(p, a.w_in, a.w_out, st, di.max_smem_optin);
  if (rc != 0) return fail(FGMS_ERR_CUDA, "expert_layer_kernel: %s (%d)", cudaGetErrorString(cudaGetLastError()), rc);
  return check_launch("expert_layer_kernel");
}
}  // namespace

extern "C" {

size_t fgms_b200_expert_layer_workspace_bytes(int tokens, int experts, int top_k, int hidden, int out_width) {
  if (tokens < 1 || tokens > fgms::EL_MAX_TOKENS || experts < 1 || experts > fgms::EL_MAX_EXPERTS || top_k < 1 || top_k > fgms::EL_MAX_TOP_K || hidden < 1 || out_width < 1)
    return 0;
  return fgms::expert_space(tokens, experts, top_k, hidden, out_width).total;
}

int fgms_b200_expert_layer(const fgms_b200_expert_layer_args* args, void* stream) {
  TraceRange trace_range("fgms_b200_expert_layer");
  if (!args) return fail(FGMS_ERR_INVALID_ARG, "null pointer");
  return run_expert_layer(*args, static_cast<cudaStream_t>(stream));
}

int fgms_b200_grouped_i8_fwd(const int8_t* codes, int64_t codes_pitch, const float* code_scale, const int8_t* kernel, int64_t kernel_pitch,
                             const float* kernel_scale, void* out, const int32_t* kpos, int n_rows, int c_in, int c_out, int groups, int dtype,
                             int zero_rest, void* workspace, size_t workspace_bytes, void* stream) {
  TraceRange trace_range("fgms_b200_grouped_i8_fwd");
  return run_grouped_i8(codes, codes_pitch, code_scale, kernel, kernel_pitch, kernel_scale, out, kpos, n_rows, c_in, c_out, groups, dtype, zero_rest, workspace,
                        workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t fgms_b200_grouped_i8_workspace_bytes(const int8_t* codes, int64_t codes_pitch, const int8_t* kernel, int64_t kernel_pitch, int n_rows, int c_in, int c_out,
                                            int groups) {
  if (n_rows < 1 || c_in < 1 || c_out < 1 || groups < 1) return 0;
  return i8_copies(RowSpan{codes, n_rows, codes_pitch, c_in, 1}, RowSpan{kernel, (int64_t)groups * c_out, kernel_pitch, c_in, 1}).total;
}

int fgms_b200_dropout(const fgms_b200_dropout_args* args, void* stream) {
  TraceRange trace_range("fgms_b200_dropout");
  if (!args) return fail(FGMS_ERR_INVALID_ARG, "null pointer");
  return run_dropout(*args, false, static_cast<cudaStream_t>(stream));
}

int fgms_b200_dropout_bwd(const fgms_b200_dropout_args* args, void* stream) {
  TraceRange trace_range("fgms_b200_dropout_bwd");
  if (!args) return fail(FGMS_ERR_INVALID_ARG, "null pointer");
  return run_dropout(*args, true, static_cast<cudaStream_t>(stream));
}

int fgms_b200_rms_norm(const fgms_b200_rms_norm_args* args, void* stream) {
  TraceRange trace_range("fgms_b200_rms_norm");
  if (!args) return fail(FGMS_ERR_INVALID_ARG, "null pointer");
  return run_rms_norm(*args, true, static_cast<cudaStream_t>(stream));
}

size_t fgms_b200_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
  DeviceInfo di;
  if (rows < 1 || width < 1 || width > fgms::NORM_MAX_WIDTH || device_info(&di) != FGMS_OK) return 0;
  return (size_t)fgms::norm_grad_cut(rows, (int)width, di.sms).blocks * (size_t)width * 4;
}

int fgms_b200_rms_norm_bwd(const fgms_b200_rms_norm_bwd_args* args, void* stream) {
  TraceRange trace_range("fgms_b200_rms_norm_bwd");
  if (!args) return fail(FGMS_ERR_INVALID_ARG, "null pointer");
  return run_rms_norm_bwd(*args, static_cast<cudaStream_t>(stream));
}

int fgms_b200_quantize_rows(const void* x, int64_t x_pitch, int8_t* codes, int64_t codes_pitch, float* scale, int64_t rows, int64_t width, int dtype, void* stream) {
  TraceRange trace_range("fgms_b200_quantize_rows");
  if (rows > 0 && !scale) return fail(FGMS_ERR_INVALID_ARG, "scale: null pointer");
  fgms_b200_rms_norm_args a = {};
  a.x = x;
  a.x_pitch = x_pitch;
  a.out = codes;
  a.out_pitch = codes_pitch;
  a.scale = scale;
  a.rows = rows;
  a.width = width;
  a.dtype = a.weight_dtype = dtype;
  return run_rms_norm(a, false, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
