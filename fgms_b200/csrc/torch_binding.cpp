// PyTorch side of the library: the operator calls and the autograd function as a CPython extension module
// (fgms_b200._native) over the C ABI of libfgms_b200.so.
//
// Argument checks, the choice of the current stream and the kernel launches of a call are a few microseconds of host
// time here; the same steps in Python took 15-20 us per call (20 us for a forward of a few hundred voxels whose
// kernel runs 6 us; 56 us per layer and pass through the autograd engine), which is what bounded every layer of up to
// about a hundred thousand voxels.  Error types are those of the reference's binding: ValueError for what pybind11
// maps from std::invalid_argument, TypeError for an argument that is no tensor, RuntimeError for a CUDA failure.
#include <array>
#include <atomic>
#include <vector>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <pybind11/pybind11.h>

#include "../../include/fgms_b200.h"

namespace {

using at::Tensor;

void check_status(int rc) {
  if (rc == FGMS_OK) return;
  const char* msg = fgms_b200_last_error();
  if (rc == FGMS_ERR_CHANNEL_MISMATCH || rc == FGMS_ERR_INVALID_ARG || rc == FGMS_ERR_UNSUPPORTED || rc == FGMS_ERR_WORKSPACE)
    TORCH_CHECK_VALUE(false, msg);
  TORCH_CHECK(false, "fgms_b200 error ", rc, ": ", msg);
}

void check_feat(const char* name, const Tensor& t, int64_t dim) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", dim, " dimensions, got ", t.dim());
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}
void check_feat(const char* name, const Tensor& t, int64_t dim, const Tensor& like) {
  check_feat(name, t, dim);
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type(), name, " must have dtype ", like.scalar_type(), ", got ", t.scalar_type());
}
void check_index(const char* name, const Tensor& t, const Tensor& like, int64_t min_len) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt, name, " must be an int32 tensor");
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), name, " must live on ", like.device());
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK_VALUE(t.numel() >= min_len, name, " needs at least ", min_len, " entries, got ", t.numel());
}

struct Arith { int dtype, math; };
Arith arith(const Tensor& t, bool arch80) {
  if (t.scalar_type() == at::kHalf) return {FGMS_DTYPE_F16, FGMS_MATH_F16};
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "unsupported feature dtype ", t.scalar_type(), ": the operator takes float16 or float32");
  return {FGMS_DTYPE_F32, arch80 ? FGMS_MATH_TF32 : FGMS_MATH_FP32};
}

void* ptr(const Tensor& t) { return t.numel() > 0 ? t.data_ptr() : nullptr; }
const int32_t* iptr(const Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// checks shared by every pass over a pair list; returns k_vol
int check_common(const Tensor& feats, const Tensor& kernel, const Tensor& kpos, const Tensor& in_map, const Tensor& out_map) {
  check_feat("in_feats", feats, 2);
  check_feat("kernel", kernel, 3, feats);
  const int64_t k_vol = kernel.size(0);
  check_index("kpos", kpos, feats, k_vol + 1);
  check_index("in_map", in_map, feats, 0);
  check_index("out_map", out_map, feats, 0);
  TORCH_CHECK_VALUE(in_map.numel() == out_map.numel(), "in_map and out_map differ in length");
  return (int)k_vol;
}

void fusion_fwd(const Tensor& in_feats, const Tensor& kernel, int64_t sum_nnz, const Tensor& out, const Tensor& kpos,
                const Tensor* qkpos, const Tensor& in_map, const Tensor& out_map, bool separate_mid, bool arch80) {
  const int k_vol = check_common(in_feats, kernel, kpos, in_map, out_map);
  check_feat("out_feats", out, 2, in_feats);
  if (qkpos) check_index("qkpos", *qkpos, in_feats, k_vol + 1);
  TORCH_CHECK_VALUE(out.size(1) == kernel.size(2), "out_feats width differs from the kernel's output channels");
  const Arith a = arith(in_feats, arch80);
  c10::cuda::CUDAGuard guard(in_feats.device());
  check_status(fgms_b200_fusion_fwd(ptr(in_feats), ptr(kernel), ptr(out), iptr(kpos), qkpos ? iptr(*qkpos) : nullptr, iptr(in_map),
                                    iptr(out_map), in_map.numel(), (int)in_feats.size(0), (int)out.size(0), (int)in_feats.size(1),
                                    (int)kernel.size(1), (int)kernel.size(2), k_vol, sum_nnz, a.dtype, a.math, separate_mid,
                                    stream_of(in_feats)));
}

void seq_fwd(const Tensor& in_feats, const Tensor& kernel, int64_t sum_nnz, const Tensor& out, const Tensor& kernel_nnz,
             const Tensor& kpos, const Tensor& in_map, const Tensor& out_map, bool separate_mid, bool arch80) {
  const int k_vol = check_common(in_feats, kernel, kpos, in_map, out_map);
  check_feat("out_feats", out, 2, in_feats);
  TORCH_CHECK_VALUE(kernel_nnz.scalar_type() == at::kInt, "kernel_nnz must be an int32 tensor");
  TORCH_CHECK_VALUE(!kernel_nnz.is_cuda(), "kernel_nnz must be a CPU tensor");
  TORCH_CHECK_VALUE(kernel_nnz.is_contiguous(), "kernel_nnz must be contiguous");
  TORCH_CHECK_VALUE(kernel_nnz.numel() >= k_vol, "kernel_nnz needs at least ", k_vol, " entries, got ", kernel_nnz.numel());
  TORCH_CHECK_VALUE(out.size(1) == kernel.size(2), "out_feats width differs from the kernel's output channels");
  const Arith a = arith(in_feats, arch80);
  c10::cuda::CUDAGuard guard(in_feats.device());
  check_status(fgms_b200_seq_fwd(ptr(in_feats), ptr(kernel), ptr(out), kernel_nnz.data_ptr<int32_t>(), iptr(kpos), iptr(in_map),
                                 iptr(out_map), in_map.numel(), (int)in_feats.size(0), (int)out.size(0), (int)in_feats.size(1),
                                 (int)kernel.size(1), (int)kernel.size(2), k_vol, sum_nnz, a.dtype, a.math, separate_mid,
                                 stream_of(in_feats)));
}

// fp32 sums of an fp16 weight gradient that has no single-launch form (or was asked for in fp32 sums): from PyTorch's
// caching allocator, so that calls on different streams or threads never share one
Tensor wgrad_workspace(const Tensor& kernel_grad, const Arith& a, bool fp32_sums) {
  if (a.dtype != FGMS_DTYPE_F16) return {};
  const int c_in = (int)kernel_grad.size(1), c_out = (int)kernel_grad.size(2), k_vol = (int)kernel_grad.size(0);
  if (!fp32_sums && k_vol >= 1 && fgms_b200_kernel_family(2, c_in, c_out, k_vol, a.dtype, a.math) == 1) return {};
  const int64_t n = std::max<int64_t>((int64_t)(fgms_b200_wgrad_workspace_bytes(c_in, c_out, k_vol, a.dtype) / 4), 64);
  return at::empty({n}, kernel_grad.options().dtype(at::kFloat));
}

// The same for both gradients in one call: also where the library is faster with one.  A call whose pointers are not 16-byte aligned
// gets none, nor one for which there is no memory, as it has another way without.
Tensor bwd_workspace(const void* grad_out, const void* feats, const void* kernel, const void* in_grad, const Tensor& kernel_grad, int64_t pairs,
                     const Arith& a, bool fp32_sums) {
  if (const Tensor ws = wgrad_workspace(kernel_grad, a, fp32_sums); ws.defined() || a.dtype != FGMS_DTYPE_F16) return ws;
  const int c_in = (int)kernel_grad.size(1), c_out = (int)kernel_grad.size(2), k_vol = (int)kernel_grad.size(0);
  const size_t bytes = fgms_b200_bwd_workspace_bytes(pairs, c_in, c_out, k_vol, a.dtype, a.math);
  uintptr_t at = 0;
  for (const void* p : {grad_out, feats, kernel, in_grad, (const void*)kernel_grad.data_ptr()}) at |= reinterpret_cast<uintptr_t>(p);
  if (bytes == 0 || (at & 15) != 0) return {};
  try {
    return at::empty({(int64_t)(bytes / 4)}, kernel_grad.options().dtype(at::kFloat));
  } catch (const c10::OutOfMemoryError&) {
    return {};
  }
}

void bwd(const Tensor& grad_out, const Tensor& in_feats, const Tensor& kernel, int64_t sum_nnz, const Tensor& in_grad,
         const Tensor& kernel_grad, const Tensor& kpos, const Tensor* qkpos, const Tensor& in_map, const Tensor& out_map,
         bool separate_mid, bool arch80, bool fp32_sums) {
  const int k_vol = check_common(in_feats, kernel, kpos, in_map, out_map);
  check_feat("out_feats_grad", grad_out, 2, in_feats);
  check_feat("in_feats_grad", in_grad, 2, in_feats);
  check_feat("kernel_grad", kernel_grad, 3, in_feats);
  if (in_feats.size(1) == kernel.size(1)) {  // a channel mismatch is the library's own error below
    TORCH_CHECK_VALUE(in_grad.sizes() == in_feats.sizes() && kernel_grad.sizes() == kernel.sizes(),
                      "gradient buffers must have the shapes of in_feats and kernel");
    TORCH_CHECK_VALUE(grad_out.size(1) == kernel.size(2), "out_feats_grad width differs from the kernel's output channels");
  }
  const Arith a = arith(in_feats, arch80);
  c10::cuda::CUDAGuard guard(in_feats.device());
  const Tensor ws = in_feats.size(1) == kernel.size(1)
                        ? bwd_workspace(ptr(grad_out), ptr(in_feats), ptr(kernel), ptr(in_grad), kernel_grad, in_map.numel(), a, fp32_sums)
                        : Tensor();
  check_status(fgms_b200_bwd(ptr(grad_out), ptr(in_feats), ptr(kernel), ptr(in_grad), ptr(kernel_grad), iptr(kpos),
                             qkpos ? iptr(*qkpos) : nullptr, iptr(in_map), iptr(out_map), in_map.numel(), (int)in_feats.size(0),
                             (int)grad_out.size(0), (int)in_feats.size(1), (int)kernel.size(1), (int)kernel.size(2), k_vol, sum_nnz,
                             a.dtype, a.math, separate_mid, ws.defined() ? ws.data_ptr() : nullptr,
                             ws.defined() ? (size_t)ws.numel() * 4 : 0, stream_of(in_feats)));
}

// ---------------------------------------------------------------------------------------------
// autograd
// ---------------------------------------------------------------------------------------------
// backend.WGRAD_FP32_SUMS.  A backward follows the switch of its own time, not of the forward's; it runs on a thread of the
// autograd engine without the GIL, so the switch is kept here and the module's attribute reads and sets it.
std::atomic<bool> g_fp32_sums{false};

size_t bytes_of(const Tensor& t) { return (size_t)t.numel() * t.element_size(); }

struct SparseConv : torch::autograd::Function<SparseConv> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& feats_, const Tensor& weight_, const Tensor& kpos,
                        const Tensor& imap, const Tensor& omap, int64_t n_out, bool arch80) {
    const Tensor feats = feats_.contiguous(), weight = weight_.contiguous();
    TORCH_CHECK_VALUE(feats.is_cuda(), "in_feats must be a CUDA tensor");
    TORCH_CHECK_VALUE(weight.dim() == 3, "kernel must have 3 dimensions, got ", weight.dim());
    c10::cuda::CUDAGuard guard(feats.device());
    Tensor out = at::empty({n_out, weight.size(2)}, feats.options().requires_grad(false));
    check_status(fgms_b200_zero2(ptr(out), bytes_of(out), nullptr, 0, stream_of(feats)));
    fusion_fwd(feats, weight, 0, out, kpos, nullptr, imap, omap, false, arch80);
    ctx->save_for_backward({feats, weight, kpos, imap, omap});
    ctx->saved_data["arch80"] = arch80;
    return out;
  }

  // Only the gradients that something needs are computed: the first layer of a network has no input gradient, a
  // frozen layer no weight gradient.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &feats = saved[0], &weight = saved[1], &kpos = saved[2], &imap = saved[3], &omap = saved[4];
    const bool arch80 = ctx->saved_data["arch80"].toBool();
    const Tensor grad_out = grads[0].contiguous();
    const bool need_in = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    // saved tensors come back through whatever hooks were installed when they were saved: as good as new arguments
    const int k_vol = check_common(feats, weight, kpos, imap, omap);
    check_feat("out_feats_grad", grad_out, 2, feats);
    TORCH_CHECK_VALUE(feats.size(1) == weight.size(1), "Input feature size and kernel size mismatch");
    TORCH_CHECK_VALUE(grad_out.size(1) == weight.size(2), "out_feats_grad width differs from the kernel's output channels");
    c10::cuda::CUDAGuard guard(feats.device());
    void* st = stream_of(feats);
    Tensor in_grad, w_grad;
    if (need_in) in_grad = at::empty_like(feats);
    if (need_w) w_grad = at::empty_like(weight);
    const Arith a = arith(feats, arch80);
    const int n_in = (int)feats.size(0), n_out = (int)grad_out.size(0), c_in = (int)weight.size(1), c_out = (int)weight.size(2);
    check_status(fgms_b200_zero2(need_in ? ptr(in_grad) : nullptr, need_in ? bytes_of(in_grad) : 0, need_w ? ptr(w_grad) : nullptr,
                                 need_w ? bytes_of(w_grad) : 0, st));
    if (need_in && need_w) {  // in one call, which lets them run side by side
      const Tensor ws = bwd_workspace(ptr(grad_out), ptr(feats), ptr(weight), ptr(in_grad), w_grad, imap.numel(), a,
                                      g_fp32_sums.load(std::memory_order_relaxed));
      check_status(fgms_b200_bwd(ptr(grad_out), ptr(feats), ptr(weight), ptr(in_grad), ptr(w_grad), iptr(kpos), nullptr, iptr(imap),
                                 iptr(omap), imap.numel(), n_in, n_out, c_in, c_in, c_out, k_vol, 0, a.dtype, a.math, 0,
                                 ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() * 4 : 0, st));
    } else if (need_in) {
      check_status(fgms_b200_dgrad(ptr(grad_out), ptr(weight), ptr(in_grad), iptr(kpos), iptr(imap), iptr(omap), imap.numel(), n_in,
                                   n_out, c_in, c_out, k_vol, a.dtype, a.math, st));
    } else if (need_w) {
      const Tensor ws = wgrad_workspace(w_grad, a, g_fp32_sums.load(std::memory_order_relaxed));
      check_status(fgms_b200_wgrad(ptr(feats), ptr(grad_out), ptr(w_grad), iptr(kpos), iptr(imap), iptr(omap), imap.numel(), n_in,
                                   n_out, c_in, c_out, k_vol, a.dtype, a.math, ws.defined() ? ws.data_ptr() : nullptr,
                                   ws.defined() ? (size_t)ws.numel() * 4 : 0, 1, st));
    }
    return {in_grad, w_grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------
// a stack of layers as one node
// ---------------------------------------------------------------------------------------------
// A node per layer costs 14 us of the engine's host time on top of its launches, and a fill of its own for the output and for the
// gradients: 1100 us for the 25 layers of an encoder-decoder on 8 k voxels whose kernels run 500 us.  Here the layers' values lie in one
// allocation, their gradients in another, each cleared by one launch, and the backward is a loop.  The arithmetic is the one of
// a node per layer: every layer adds into zeros, a skip connection and its gradient are sums rounded once.
//
// A node per layer needs less memory: it hands back its input and its output's gradient as the backward goes on.  So beyond STACK_BYTES
// of values, and where there is no memory for one allocation, values and gradients are allocated and cleared one by one and dropped in the
// same way.  Training steps of the 25 layers, peaks above what is there before: 120 k voxels, 59 MB of values, a node per layer 66 MB, two
// allocations 123; 240 k voxels, 113 MB, 129 MB a node per layer and one by one, 231 in two allocations.  By then the device is
// busy for longer than the further allocations and launches take the host: 1970 us a node per layer, 1080-1150 one by one, 965 in two.
//
// Value 0 is the input, value l + 1 what layer l produces.
struct StackLayer { int64_t src, skip /* -1: none */, map, n_in, n_out; };
using StackPlan = std::vector<int64_t>;  // StackLayer by StackLayer
constexpr int64_t STACK_FIELDS = 5;
constexpr int64_t STACK_BYTES = 64 << 20;
StackLayer layer_of(const StackPlan& plan, size_t l) {
  const int64_t* f = plan.data() + l * STACK_FIELDS;
  return {f[0], f[1], f[2], f[3], f[4]};
}

// What every layer's own call would accept, and what one node can hold: each value but the last is used, by one layer at most.
// False: the caller runs layer by layer, and meets its errors there.
bool stack_suits(const Tensor& feats, at::TensorList weights, at::TensorList maps, const StackPlan& plan, bool arch80) {
  const size_t n = weights.size();
  const auto dtype = feats.scalar_type();
  if (n == 0 || plan.size() != n * STACK_FIELDS || maps.size() % 3 != 0) return false;
  if (!feats.is_cuda() || feats.dim() != 2 || !feats.is_contiguous() || (dtype != at::kHalf && dtype != at::kFloat)) return false;
  auto aligned = [](const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; };
  if (feats.numel() == 0 || !aligned(feats)) return false;
  for (const Tensor& m : maps)
    if (m.scalar_type() != at::kInt || m.device() != feats.device() || !m.is_contiguous() || m.requires_grad()) return false;
  struct Value { int64_t rows, width; int convs, skips; };
  std::vector<Value> value(1, {feats.size(0), feats.size(1), 0, 0});
  value.reserve(n + 1);
  for (size_t l = 0; l < n; ++l) {
    const StackLayer s = layer_of(plan, l);
    const Tensor& w = weights[l];
    const int64_t known = (int64_t)value.size();
    if (w.scalar_type() != dtype || w.device() != feats.device() || w.dim() != 3 || !w.is_contiguous() || w.numel() == 0 || !aligned(w)) return false;
    if (s.src < 0 || s.src >= known || s.skip >= known || s.map < 0 || 3 * s.map + 2 >= (int64_t)maps.size() || s.n_out < 1) return false;
    const Tensor &kpos = maps[3 * s.map], &imap = maps[3 * s.map + 1], &omap = maps[3 * s.map + 2];
    Value& from = value[s.src];
    if (from.rows != s.n_in || from.width != w.size(1) || kpos.numel() != w.size(0) + 1 || imap.numel() != omap.numel()) return false;
    if (from.convs++ > 0) return false;
    value.push_back({s.n_out, w.size(2), 0, 0});
    if (s.skip >= 0) {
      Value& add = value[s.skip];
      if (add.rows != s.n_out || add.width != w.size(2)) return false;
      ++add.skips;
    }
  }
  for (size_t v = 1; v < n; ++v)
    if (value[v].convs + value[v].skips == 0) return false;
  return true;
}

struct SparseStack : torch::autograd::Function<SparseStack> {
  // What the node keeps, in elements: the values that layers 0 .. n - 2 produce (slots 1 .. n - 1) and, where the input's few fp16
  // channels are padded to a multiple of 16 (8-byte rows cannot be gathered in 16-byte pieces and would run on the CUDA cores: 4 -> 32
  // on 84 k pairs 16.6 / 45 us forward / weight gradient, padded 4.9 / 6.2), the padded input (slot 0) and the weights that go with it (slot n).
  struct Layout {
    std::vector<int64_t> count, at;  // of a slot; its place in a block of all of them, from a 256-byte boundary
    int64_t end = 0;                 // of that block
    int64_t pad = 0;                 // channels of the padded input, 0: as it is
    template <typename Kept>
    Layout(const Tensor& feats, at::TensorList kernels, const StackPlan& plan, bool padding, Kept kept) {
      const size_t n = kernels.size();
      count.resize(n + 1);
      at.resize(n + 1);
      for (size_t l = 0; l + 1 < n; ++l)
        if (kept(l + 1)) count[l + 1] = layer_of(plan, l).n_out * kernels[l].size(2);
      const Tensor* reader = nullptr;  // the layer of the input
      padding = padding && feats.scalar_type() == at::kHalf && feats.size(1) % 16 != 0 && feats.size(1) <= 256;
      for (size_t l = 0; padding && l < n; ++l) {
        padding = layer_of(plan, l).skip != 0;
        if (layer_of(plan, l).src == 0) reader = &kernels[l];
      }
      if (padding && reader && reader->size(2) % 16 == 0 && reader->size(2) <= 256) {
        pad = (feats.size(1) + 15) / 16 * 16;
        count[0] = feats.size(0) * pad;
        count[n] = reader->size(0) * pad * reader->size(2);
      }
      for (size_t i = 0; i <= n; ++i) {
        at[i] = end;
        end += (count[i] + 127) / 128 * 128;
      }
    }
  };
  // The slots of a layout: in one block, or by themselves (each until it is dropped).
  struct Slots {
    const Layout& layout;
    at::TensorOptions options;
    Tensor block;
    std::vector<Tensor> own;
    Slots(const Layout& l, const Tensor& like) : layout(l), options(like.options().requires_grad(false)) {}
    bool apart() const { return !own.empty(); }
    // a block where there is memory for one and `may` says so
    void take(bool may) {
      if (may) {
        try {
          block = at::empty({layout.end}, options);
          return;
        } catch (const c10::OutOfMemoryError&) {
        }
      }
      own.resize(layout.count.size());
    }
    const Tensor& make(size_t i) { return own[i] = at::empty({layout.count[i]}, options); }
    void drop(size_t i) { if (apart()) own[i].reset(); }
    void* of(size_t i) const {
      return apart() ? own[i].data_ptr() : static_cast<uint8_t*>(block.data_ptr()) + layout.at[i] * block.element_size();
    }
  };
  // the input and its layer's weights with further channels of zeros, into cleared slots
  static void pad_input(const Slots& slots, const Tensor& feats, const Tensor& w, int dtype, void* st) {
    const int64_t pad = slots.layout.pad, c_in = feats.size(1);
    check_status(fgms_b200_copy_rows_f16(ptr(feats), c_in, dtype, slots.of(0), pad, feats.size(0), (int)c_in, st));
    check_status(fgms_b200_copy_rows_f16(ptr(w), c_in * w.size(2), dtype, slots.of(slots.layout.at.size() - 1), pad * w.size(2), w.size(0), (int)(c_in * w.size(2)), st));
  }

  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& feats, at::TensorList weights, at::TensorList maps,
                        const StackPlan& plan, bool arch80) {
    const size_t n = weights.size();
    c10::cuda::CUDAGuard guard(feats.device());
    void* st = stream_of(feats);
    const Arith a = arith(feats, arch80);
    const Layout in(feats, weights, plan, true, [](size_t) { return true; });
    Slots values(in, feats);
    values.take(in.end * (int64_t)feats.element_size() <= STACK_BYTES);
    Tensor out = at::empty({layer_of(plan, n - 1).n_out, weights[n - 1].size(2)}, values.options);
    auto cleared = [&](const Tensor& t) { check_status(fgms_b200_zero2(ptr(t), bytes_of(t), nullptr, 0, st)); };
    if (values.apart()) cleared(out);
    else check_status(fgms_b200_zero2(ptr(values.block), bytes_of(values.block), ptr(out), bytes_of(out), st));
    auto make = [&](size_t i) {
      if (values.apart()) cleared(values.make(i));
    };
    auto value = [&](int64_t v) -> void* {
      if (v == 0) return in.pad ? values.of(0) : feats.data_ptr();
      return v == (int64_t)n ? out.data_ptr() : values.of(v);
    };
    for (size_t l = 0; l < n; ++l) {
      const StackLayer s = layer_of(plan, l);
      const Tensor &w = weights[l], &imap = maps[3 * s.map + 1];
      const bool padded = s.src == 0 && in.pad;
      if (padded) {
        make(0);
        make(n);
        pad_input(values, feats, w, a.dtype, st);
      }
      if (l + 1 < n) make(l + 1);
      const int c_in = padded ? (int)in.pad : (int)w.size(1);
      check_status(fgms_b200_fusion_fwd(value(s.src), padded ? values.of(n) : ptr(w), value(l + 1), iptr(maps[3 * s.map]), nullptr, iptr(imap),
                                        iptr(maps[3 * s.map + 2]), imap.numel(), (int)s.n_in, (int)s.n_out, c_in, c_in, (int)w.size(2), (int)w.size(0), 0,
                                        a.dtype, a.math, 0, st));
      if (s.skip >= 0) check_status(fgms_b200_add(value(l + 1), value(s.skip), s.n_out * w.size(2), a.dtype, st));
      if (padded) {  // made again for the backward
        values.drop(0);
        values.drop(n);
      }
    }
    torch::autograd::variable_list saved;
    saved.reserve(2 + n + maps.size());
    saved.push_back(feats);
    saved.push_back(values.block);
    saved.insert(saved.end(), weights.begin(), weights.end());
    saved.insert(saved.end(), maps.begin(), maps.end());
    ctx->save_for_backward(std::move(saved));
    if (values.apart()) ctx->saved_data["values"] = values.own;
    ctx->saved_data["plan"] = plan;
    ctx->saved_data["arch80"] = arch80;
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const StackPlan plan = ctx->saved_data["plan"].toIntVector();
    const bool arch80 = ctx->saved_data["arch80"].toBool();
    const size_t n = plan.size() / STACK_FIELDS;
    const Tensor& feats = saved[0];
    const at::TensorList weights(saved.data() + 2, n), maps(saved.data() + 2 + n, saved.size() - 2 - n);
    TORCH_CHECK_VALUE(stack_suits(feats, weights, maps, plan, arch80), "saved tensors of the stack are not the ones it was run with");
    Tensor grad_out = grads[0].contiguous();
    check_feat("out_feats_grad", grad_out, 2, feats);
    if (reinterpret_cast<uintptr_t>(grad_out.data_ptr()) & 15) grad_out = grad_out.clone();
    c10::cuda::CUDAGuard guard(feats.device());
    void* st = stream_of(feats);
    const Arith a = arith(feats, arch80);
    TORCH_CHECK_VALUE(grad_out.size(0) == layer_of(plan, n - 1).n_out && grad_out.size(1) == weights[n - 1].size(2),
                      "out_feats_grad has another shape than the output");
    const Layout in(feats, weights, plan, true, [](size_t) { return true; });
    Slots values(in, feats);
    values.block = saved[1];
    if (const auto kept = ctx->saved_data.find("values"); kept != ctx->saved_data.end()) {
      // the last backward hands them back on the way
      values.own = kept->second.toTensorVector();
      if (!torch::autograd::get_current_graph_task_keep_graph()) ctx->saved_data.erase(kept);
    } else {
      const Tensor& block = values.block;
      TORCH_CHECK_VALUE(block.defined() && block.scalar_type() == feats.scalar_type() && block.device() == feats.device() && block.is_contiguous() &&
                        block.numel() == in.end && (reinterpret_cast<uintptr_t>(block.data_ptr()) & 15) == 0, "saved values of the stack are not the ones it was run with");
    }
    // gradients that something needs: a value's, if a weight before it or the input needs one
    std::vector<char> need(n + 1, 0), need_w(n);
    need[0] = ctx->needs_input_grad(0);
    for (size_t l = 0; l < n; ++l) {
      const StackLayer s = layer_of(plan, l);
      need_w[l] = ctx->needs_input_grad(1 + l);
      need[l + 1] = need_w[l] || need[s.src] || (s.skip >= 0 && need[s.skip]);
    }
    const Layout out(feats, weights, plan, false, [&](size_t v) { return need[v] != 0; });
    torch::autograd::variable_list result(1 + n + maps.size() + 2);
    Slots g_values(out, feats);
    g_values.take(!values.apart());
    Tensor g_input;
    auto make_g_input = [&] { return at::empty({feats.size(0), in.pad ? in.pad : feats.size(1)}, values.options); };
    if (!g_values.apart()) {  // otherwise each when it is first used
      std::vector<void*> clear;
      std::vector<size_t> bytes;
      auto add = [&](const Tensor& t) { clear.push_back(ptr(t)); bytes.push_back(bytes_of(t)); };
      add(g_values.block);
      if (need[0]) add(g_input = make_g_input());
      for (size_t l = 0; l < n; ++l)
        if (need_w[l]) add(result[1 + l] = at::empty_like(weights[l]));
      check_status(fgms_b200_zero_list(clear.data(), bytes.data(), (int)clear.size(), st));
    }
    auto cleared = [&](const Tensor& t) { check_status(fgms_b200_zero2(ptr(t), bytes_of(t), nullptr, 0, st)); };
    auto value = [&](int64_t v) -> void* { return v == 0 && !in.pad ? feats.data_ptr() : values.of(v); };
    auto grad = [&](int64_t v) -> void* {
      if (v == (int64_t)n) return grad_out.data_ptr();
      if (v == 0) {
        if (!g_input.defined()) cleared(g_input = make_g_input());
        return g_input.data_ptr();
      }
      if (g_values.apart() && !g_values.own[v].defined()) cleared(g_values.make(v));
      return g_values.of(v);
    };
    std::vector<std::vector<int64_t>> added(n + 1);  // values whose gradient is part of a value's, through a skip connection
    auto finish = [&](int64_t v, int64_t count) {    // its layer's input gradient is in it
      for (int64_t from : added[v]) {
        check_status(fgms_b200_add(grad(v), grad(from), count, a.dtype, st));
        if (from < (int64_t)n) g_values.drop(from);
      }
    };
    const bool fp32_sums = g_fp32_sums.load(std::memory_order_relaxed);
    // both gradients of a layer
    auto layer = [&](size_t l, const StackLayer& s) {
      const Tensor &w = weights[l], &imap = maps[3 * s.map + 1];
      const int32_t *kpos = iptr(maps[3 * s.map]), *im = iptr(imap), *om = iptr(maps[3 * s.map + 2]);
      const int c_in = (int)w.size(1), c_out = (int)w.size(2), k_vol = (int)w.size(0), n_in = (int)s.n_in, n_out = (int)s.n_out;
      if (need_w[l] && !result[1 + l].defined()) cleared(result[1 + l] = at::empty_like(w));
      if (s.src == 0 && in.pad) {
        const int pad = (int)in.pad;
        if (values.apart()) {
          cleared(values.make(0));
          cleared(values.make(n));
          pad_input(values, feats, w, a.dtype, st);
        }
        if (need_w[l]) {  // fp32 sums, of which the rows of the real channels are rounded
          const Tensor sums = at::empty({(int64_t)k_vol * pad * c_out}, w.options().dtype(at::kFloat).requires_grad(false));
          check_status(fgms_b200_wgrad(value(0), grad(l + 1), nullptr, kpos, im, om, imap.numel(), n_in, n_out, pad, c_out, k_vol, a.dtype, a.math,
                                       sums.data_ptr(), bytes_of(sums), 0, st));
          check_status(fgms_b200_copy_rows_f16(sums.data_ptr(), pad * c_out, FGMS_DTYPE_F32, result[1 + l].data_ptr(), c_in * c_out, k_vol, c_in * c_out, st));
        }
        if (need[0])
          check_status(fgms_b200_dgrad(grad(l + 1), values.of(n), grad(0), kpos, im, om, imap.numel(), n_in, n_out, pad, c_out, k_vol, a.dtype, a.math, st));
        return;
      }
      const Tensor ws = !need_w[l] ? Tensor()
                        : need[s.src] ? bwd_workspace(grad(l + 1), value(s.src), ptr(w), grad(s.src), result[1 + l], imap.numel(), a, fp32_sums)
                                      : wgrad_workspace(result[1 + l], a, fp32_sums);
      void* ws_ptr = ws.defined() ? ws.data_ptr() : nullptr;
      const size_t ws_bytes = ws.defined() ? bytes_of(ws) : 0;
      if (need[s.src] && need_w[l])
        check_status(fgms_b200_bwd(grad(l + 1), value(s.src), ptr(w), grad(s.src), result[1 + l].data_ptr(), kpos, nullptr, im, om, imap.numel(), n_in,
                                   n_out, c_in, c_in, c_out, k_vol, 0, a.dtype, a.math, 0, ws_ptr, ws_bytes, st));
      else if (need[s.src])
        check_status(fgms_b200_dgrad(grad(l + 1), ptr(w), grad(s.src), kpos, im, om, imap.numel(), n_in, n_out, c_in, c_out, k_vol, a.dtype, a.math, st));
      else if (need_w[l])
        check_status(fgms_b200_wgrad(value(s.src), grad(l + 1), result[1 + l].data_ptr(), kpos, im, om, imap.numel(), n_in, n_out, c_in, c_out, k_vol,
                                     a.dtype, a.math, ws_ptr, ws_bytes, 1, st));
    };
    for (size_t l = n; l-- > 0;) {
      const StackLayer s = layer_of(plan, l);
      if (need[l + 1]) {
        if (l + 1 < n) finish(l + 1, s.n_out * weights[l].size(2));
        layer(l, s);
        if (s.skip >= 0 && need[s.skip]) added[s.skip].push_back(l + 1);
        else if (l + 1 < n) g_values.drop(l + 1);
      }
      values.drop(s.src);  // no other layer reads it
    }
    if (need[0]) {
      finish(0, feats.numel());
      grad(0);
      result[0] = in.pad ? g_input.narrow(1, 0, feats.size(1)).contiguous() : g_input;
    }
    return result;
  }
};

// output-stationary forward into `out`; nbr is the table fgms_b200_build_neighbor_table fills
void fwd_os(const Tensor& in_feats, const Tensor& kernel, const Tensor& out, const Tensor& nbr, bool arch80, const Tensor* bias,
            bool relu, bool accumulate) {
  check_feat("in_feats", in_feats, 2);
  check_feat("kernel", kernel, 3, in_feats);
  check_feat("out_feats", out, 2, in_feats);
  TORCH_CHECK_VALUE(kernel.size(1) == in_feats.size(1), "Input feature size and kernel size mismatch");
  TORCH_CHECK_VALUE(out.size(1) == kernel.size(2), "out_feats width differs from the kernel's output channels");
  const int64_t k_vol = kernel.size(0), stride = (out.size(0) + 127) / 128 * 128;
  TORCH_CHECK_VALUE(nbr.scalar_type() == at::kInt && nbr.is_contiguous() && nbr.device() == in_feats.device() && nbr.numel() == k_vol * stride,
                    "nbr must be the contiguous int32 table build_neighbor_table returns for these sizes");
  if (bias) {
    check_feat("bias", *bias, 1, in_feats);
    TORCH_CHECK_VALUE(bias->numel() == kernel.size(2), "bias length differs from the kernel's output channels");
  }
  const Arith a = arith(in_feats, arch80);
  c10::cuda::CUDAGuard guard(in_feats.device());
  check_status(fgms_b200_fwd_output_stationary(ptr(in_feats), ptr(kernel), ptr(out), iptr(nbr), (int)in_feats.size(0), (int)out.size(0),
                                               (int)in_feats.size(1), (int)kernel.size(2), (int)k_vol, a.dtype, a.math,
                                               bias ? ptr(*bias) : nullptr, relu, accumulate, stream_of(in_feats)));
}

// ---------------------------------------------------------------------------------------------
// kernel maps
// ---------------------------------------------------------------------------------------------
struct Pyramid {
  bool fits = false;
  std::vector<int64_t> voxels;                  // per level
  std::vector<std::array<Tensor, 3>> maps;      // kpos, imap, omap
  std::vector<Tensor> out_coords;               // level 1 ..
};

// The maps of `what` (see fgms_b200_pyramid_plan) of the cloud and its coarser levels.  One wait, for the sizes (two if the
// box turns out larger than the first workspace has room for); the Python objects around the maps are made while the last
// kernel runs.
Pyramid try_pyramid(const Tensor& coords, int levels, int what) {
  TORCH_CHECK_VALUE(coords.is_cuda() && coords.scalar_type() == at::kInt && coords.dim() == 2 && coords.size(1) == 3 && coords.is_contiguous(),
                    "coords must be a contiguous CUDA int32 tensor of shape [n, 3]");
  Pyramid r;
  const int64_t n64 = coords.size(0);
  if (n64 < 1 || n64 > 0x7fffffffll / 27) return r;
  const int n = (int)n64;
  size_t bytes = fgms_b200_pyramid_workspace_bytes(n, levels, what);
  if (bytes == 0) return r;
  c10::cuda::CUDAGuard guard(coords.device());
  void* st = stream_of(coords);
  const auto ints = coords.options();
  const int n_maps = ((what & 1) ? levels : 0) + ((what & 2) ? levels - 1 : 0) + ((what & 4) ? levels - 1 : 0);
  const Tensor host = at::empty({64}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
  const int32_t* sizes = host.data_ptr<int32_t>();
  Tensor ws, kpos;
  std::vector<int32_t*> coord_ptrs;
  for (int attempt = 0;; ++attempt) {
    ws = Tensor();  // before the larger one
    ws = at::empty({(int64_t)bytes}, ints.dtype(at::kByte));
    if (attempt == 0) {
      kpos = at::empty({n_maps * 28}, ints);
      for (int l = 1; l < levels; ++l) {
        r.out_coords.push_back(at::empty({n64, 3}, ints));
        coord_ptrs.push_back(r.out_coords.back().data_ptr<int32_t>());
      }
    }
    int rc;
    {
      pybind11::gil_scoped_release unlock;  // this waits for the device
      rc = fgms_b200_pyramid_plan(iptr(coords), n, levels, what, kpos.data_ptr<int32_t>(), coord_ptrs.data(), ws.data_ptr(), bytes,
                                  host.data_ptr<int32_t>(), st);
    }
    check_status(rc);
    if (sizes[0] == 0) break;
    if (sizes[1] == 0 || attempt > 0) return Pyramid();
    bytes = (size_t)sizes[1] * 256;
  }
  r.fits = true;
  for (int l = 0; l < levels; ++l) r.voxels.push_back(sizes[1 + l]);
  // Both sides of a map in one allocation, each on a 256-byte boundary; a map has memory of its own, so that one that is kept does not
  // keep the others.  The device waits for the addresses only: they become tensors while it writes the maps, one TensorImpl a side
  // (13 maps of 120 k voxels: at::empty here and narrow there 112 us, so 91).
  c10::Allocator* memory = c10::cuda::CUDACachingAllocator::get();
  auto padded = [&](int j) { return ((int64_t)sizes[1 + levels + j] + 64) / 64 * 64; };
  std::vector<c10::DataPtr> flat;
  std::vector<int32_t*> in_maps, out_maps;
  flat.reserve(n_maps);
  for (int j = 0; j < n_maps; ++j) {
    flat.push_back(memory->allocate(2 * padded(j) * sizeof(int32_t)));
    in_maps.push_back(static_cast<int32_t*>(flat[j].get()));
    out_maps.push_back(in_maps[j] + padded(j));
  }
  check_status(fgms_b200_pyramid_emit(iptr(coords), n, levels, what, kpos.data_ptr<int32_t>(), coord_ptrs.data(), in_maps.data(),
                                      out_maps.data(), ws.data_ptr(), bytes, st));
  for (int j = 0; j < n_maps; ++j) {
    const c10::Storage storage(c10::Storage::use_byte_size_t(), 2 * padded(j) * sizeof(int32_t), std::move(flat[j]), memory, true);
    auto side = [&](int64_t offset) {
      Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA), caffe2::TypeMeta::Make<int32_t>());
      t.unsafeGetTensorImpl()->set_storage_offset(offset);
      t.unsafeGetTensorImpl()->set_sizes_contiguous({(int64_t)sizes[1 + levels + j]});
      return t;
    };
    const bool subm = (what & 1) && j < levels;
    r.maps.push_back({kpos.narrow(0, j * 28, subm ? 28 : 9), side(0), side(padded(j))});
  }
  for (int l = 1; l < levels; ++l) r.out_coords[l - 1] = r.out_coords[l - 1].narrow(0, 0, r.voxels[l]);
  return r;
}

// A cloud for whose bitmaps there is no memory does not fit either: the other builders need less.
Pyramid build_pyramid(const Tensor& coords, int levels, int what) {
  try {
    return try_pyramid(coords, levels, what);
  } catch (const c10::OutOfMemoryError&) {
    return Pyramid();
  }
}

// ---------------------------------------------------------------------------------------------
// products of ragged groups of rows
// ---------------------------------------------------------------------------------------------
// autograd notices that a tensor it has saved was written
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int grouped_dtype(const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return FGMS_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return FGMS_DTYPE_BF16;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "unsupported feature dtype ", t.scalar_type(),
                    ": the grouped products take float16, bfloat16 or float32");
  return FGMS_DTYPE_F32;
}

// rows [n, width] of the weights' type and device, where a row's width is the weights' dimension `side`
void check_rows(const char* name, const Tensor& t, const Tensor& weights, int side) {
  check_feat(name, t, 2, weights);
  TORCH_CHECK_VALUE(t.device() == weights.device(), name, " must live on ", weights.device());
  TORCH_CHECK_VALUE(t.size(1) == weights.size(side), name, " has ", t.size(1), " channels, the weights say ", weights.size(side));
  TORCH_CHECK_VALUE(t.size(0) <= 0x7fffffff, name, " has more than 2^31 - 1 rows");
}
void check_groups(const char* name, const Tensor& weights, const Tensor& kpos) {
  check_feat(name, weights, 3);
  check_index("kpos", kpos, weights, 0);
  TORCH_CHECK_VALUE(kpos.dim() == 1 && kpos.size(0) == weights.size(0) + 1, "kpos must have one entry more than there are groups: ",
                    weights.size(0) + 1, ", got ", kpos.numel());
  for (int d = 1; d < 3; ++d) TORCH_CHECK_VALUE(weights.size(d) <= 0x7fffffff, "more than 2^31 - 1 channels");
}

// Rows that no tensor map can describe are copied: into PyTorch's caching allocator's memory, so that calls on different streams or threads never share
// it.  Where there is none, the call has another way.
Tensor grouped_workspace(int pass, const Tensor& a, const Tensor& b, const Tensor& d, int64_t rows, const Tensor& kernel, int dtype) {
  const size_t bytes = fgms_b200_grouped_workspace_bytes(pass, ptr(a), ptr(b), ptr(d), (int)rows, (int)kernel.size(1), (int)kernel.size(2),
                                                         (int)kernel.size(0), dtype);
  if (bytes == 0) return {};
  try {
    return at::empty({(int64_t)bytes}, kernel.options().dtype(at::kByte).requires_grad(false));
  } catch (const c10::OutOfMemoryError&) {
    return {};
  }
}
void* space(const Tensor& ws) { return ws.defined() ? ws.data_ptr() : nullptr; }
size_t space_bytes(const Tensor& ws) { return ws.defined() ? (size_t)ws.numel() : 0; }

void grouped_fwd(const Tensor& in_feats, const Tensor& kernel, const Tensor& out, const Tensor& kpos, bool zero_rest) {
  check_groups("kernel", kernel, kpos);
  check_rows("in_feats", in_feats, kernel, 1);
  check_rows("out_feats", out, kernel, 2);
  TORCH_CHECK_VALUE(in_feats.size(0) == out.size(0), "in_feats and out_feats differ in rows");
  const int dtype = grouped_dtype(kernel);
  c10::cuda::CUDAGuard guard(kernel.device());
  const Tensor ws = grouped_workspace(0, in_feats, kernel, out, out.size(0), kernel, dtype);
  check_status(fgms_b200_grouped_fwd(ptr(in_feats), ptr(kernel), ptr(out), iptr(kpos), (int)out.size(0), (int)kernel.size(1), (int)kernel.size(2),
                                     (int)kernel.size(0), dtype, zero_rest, space(ws), space_bytes(ws), stream_of(kernel)));
  written(out);
}

void grouped_dgrad(const Tensor& grad_out, const Tensor& kernel, const Tensor& in_grad, const Tensor& kpos, bool zero_rest) {
  check_groups("kernel", kernel, kpos);
  check_rows("out_feats_grad", grad_out, kernel, 2);
  check_rows("in_feats_grad", in_grad, kernel, 1);
  TORCH_CHECK_VALUE(in_grad.size(0) == grad_out.size(0), "out_feats_grad and in_feats_grad differ in rows");
  const int dtype = grouped_dtype(kernel);
  c10::cuda::CUDAGuard guard(kernel.device());
  const Tensor ws = grouped_workspace(1, grad_out, kernel, in_grad, in_grad.size(0), kernel, dtype);
  check_status(fgms_b200_grouped_dgrad(ptr(grad_out), ptr(kernel), ptr(in_grad), iptr(kpos), (int)in_grad.size(0), (int)kernel.size(1),
                                       (int)kernel.size(2), (int)kernel.size(0), dtype, zero_rest, space(ws), space_bytes(ws), stream_of(kernel)));
  written(in_grad);
}

void grouped_wgrad(const Tensor& in_feats, const Tensor& grad_out, const Tensor& kernel_grad, const Tensor& kpos) {
  check_groups("kernel_grad", kernel_grad, kpos);
  check_rows("in_feats", in_feats, kernel_grad, 1);
  check_rows("out_feats_grad", grad_out, kernel_grad, 2);
  TORCH_CHECK_VALUE(in_feats.size(0) == grad_out.size(0), "in_feats and out_feats_grad differ in rows");
  const int dtype = grouped_dtype(kernel_grad);
  c10::cuda::CUDAGuard guard(kernel_grad.device());
  const Tensor ws = grouped_workspace(2, in_feats, grad_out, kernel_grad, in_feats.size(0), kernel_grad, dtype);
  check_status(fgms_b200_grouped_wgrad(ptr(in_feats), ptr(grad_out), ptr(kernel_grad), iptr(kpos), (int)in_feats.size(0), (int)kernel_grad.size(1),
                                       (int)kernel_grad.size(2), (int)kernel_grad.size(0), dtype, space(ws), space_bytes(ws), stream_of(kernel_grad)));
  written(kernel_grad);
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& feats_, const Tensor& weight_, const Tensor& kpos) {
    const Tensor feats = feats_.contiguous(), weight = weight_.contiguous();
    check_groups("weight", weight, kpos);
    check_rows("feats", feats, weight, 1);
    Tensor out = at::empty({feats.size(0), weight.size(2)}, feats.options().requires_grad(false));
    grouped_fwd(feats, weight, out, kpos, true);
    ctx->save_for_backward({feats, weight, kpos});
    return out;
  }

  // only the gradients that something needs; rows of no group have a gradient of zero
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &feats = saved[0], &weight = saved[1], &kpos = saved[2];
    const Tensor grad_out = grads[0].contiguous();
    Tensor in_grad, w_grad;
    if (ctx->needs_input_grad(0)) {
      in_grad = at::empty_like(feats);
      grouped_dgrad(grad_out, weight, in_grad, kpos, true);
    }
    if (ctx->needs_input_grad(1)) {
      w_grad = at::empty_like(weight);
      grouped_wgrad(feats, grad_out, w_grad, kpos);
    }
    if (!at::GradMode::is_enabled()) return {in_grad, w_grad, Tensor()};
    // a graph of the backward was asked for: it ends here, and says so to whoever goes through it
    for (Tensor* t : {&in_grad, &w_grad}) {
      if (!t->defined()) continue;
      t->set_requires_grad(true);
      const auto ends = std::make_shared<torch::autograd::DelayedError>("grouped_linear is not differentiable twice", 1);
      *t = (*ends)({*t})[0];
    }
    return {in_grad, w_grad, Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------
// between two layers: norm, dropout, rows in 8 bits
// ---------------------------------------------------------------------------------------------
int layer_dtype(const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return FGMS_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return FGMS_DTYPE_BF16;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "unsupported feature dtype ", t.scalar_type(), ": rows are float16, bfloat16 or float32");
  return FGMS_DTYPE_F32;
}

// rows [n, width] whose values lie side by side; the rows themselves may be apart
void check_row_values(const char* name, const Tensor& t, at::ScalarType type, const Tensor& like) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must live on ", like.device());
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must have dtype ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must have 2 dimensions, got ", t.dim());
  TORCH_CHECK_VALUE(t.size(0) == like.size(0) && t.size(1) == like.size(1), name, " is ", t.size(0), " x ", t.size(1), ", the rows are ", like.size(0), " x ",
                    like.size(1));
  TORCH_CHECK_VALUE(t.numel() == 0 || t.size(1) <= 1 || t.stride(1) == 1, name, " must have the values of a row side by side");
  TORCH_CHECK_VALUE(t.numel() == 0 || t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " has rows that overlap");
}
int64_t pitch(const Tensor& t) { return t.numel() > 0 && t.size(0) > 1 ? t.stride(0) : t.size(1); }
// one value of a type for each of `n` rows or columns
void* check_line(const char* name, const Tensor& t, at::ScalarType type, int64_t n, const Tensor& like) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must live on ", like.device());
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must have dtype ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.is_contiguous() && t.dim() == 1 && t.numel() == n, name, " must be ", n, " values side by side");
  return ptr(t);
}
int64_t* check_rng(const char* name, const Tensor* t, int64_t n, const Tensor& like) {
  TORCH_CHECK_VALUE(t != nullptr, name, " is needed where values are dropped");
  return static_cast<int64_t*>(check_line(name, *t, at::kLong, n, like));
}
// whether a probability, rounded to 16 bits, drops anything (the library refuses what is no probability)
bool drops(double p) { return !(p >= 0.0 && p * 65536.0 <= 0.5); }

struct NormCall {
  const Tensor &x, *weight, &out;
  const Tensor *residual, *sum, *scale, *rstd, *rng, *used;
  double eps, p;
};
void rms_norm(const NormCall& c) {
  const Tensor& x = c.x;
  const int dtype = layer_dtype(x);
  check_row_values("x", x, x.scalar_type(), x);
  check_row_values("out", c.out, c.scale ? at::kChar : x.scalar_type(), x);
  if (c.residual) check_row_values("residual", *c.residual, x.scalar_type(), x);
  if (c.sum) check_row_values("residual_out", *c.sum, x.scalar_type(), x);
  if (x.size(1) == 0) return;
  fgms_b200_rms_norm_args a = {};
  if (c.weight) {
    TORCH_CHECK_VALUE(c.weight->scalar_type() == x.scalar_type() || c.weight->scalar_type() == at::kFloat, "weight must have dtype ", x.scalar_type(),
                      " or float32, got ", c.weight->scalar_type());
    a.weight = check_line("weight", *c.weight, c.weight->scalar_type(), x.size(1), x);
    a.weight_dtype = layer_dtype(*c.weight);
  }
  if (c.scale) a.scale = static_cast<float*>(check_line("scale", *c.scale, at::kFloat, x.size(0), x));
  if (c.rstd) a.rstd = static_cast<float*>(check_line("rstd", *c.rstd, at::kFloat, x.size(0), x));
  const bool drop = drops(c.p);
  if (drop) {
    a.rng = check_rng("rng", c.rng, 3, x);
    if (c.used) a.rng_used = check_rng("rng_used", c.used, 2, x);
  }
  a.x = ptr(x);
  a.out = ptr(c.out);
  a.x_pitch = pitch(x);
  a.out_pitch = pitch(c.out);
  if (c.residual) a.residual = ptr(*c.residual), a.residual_pitch = pitch(*c.residual);
  if (c.sum) a.sum = ptr(*c.sum), a.sum_pitch = pitch(*c.sum);
  a.rows = x.size(0);
  a.width = x.size(1);
  a.eps = c.eps;
  a.p = c.p;
  a.dtype = dtype;
  c10::cuda::CUDAGuard guard(x.device());
  if (c.weight) check_status(fgms_b200_rms_norm(&a, stream_of(x)));
  else check_status(fgms_b200_quantize_rows(a.x, a.x_pitch, static_cast<int8_t*>(a.out), a.out_pitch, a.scale, a.rows, a.width, dtype, stream_of(x)));
  written(c.out);
  for (const Tensor* t : {c.sum, c.scale, c.rstd, drop ? c.rng : nullptr, drop ? c.used : nullptr})
    if (t) written(*t);
}

struct NormGradCall {
  const Tensor &out_grad, &weight, &rstd;
  const Tensor *sum, *x, *residual, *sum_grad, *x_grad, *residual_grad, *weight_grad, *used;  // sum, or x with residual or none
  double p;
};
void rms_norm_bwd(const NormGradCall& c) {
  TORCH_CHECK_VALUE((c.sum != nullptr) != (c.x != nullptr), "either h or x is needed");
  TORCH_CHECK_VALUE(c.x || !c.residual, "residual goes with x");
  const Tensor& h = c.x ? *c.x : *c.sum;
  fgms_b200_rms_norm_bwd_args a = {};
  a.dtype = layer_dtype(h);
  check_row_values(c.x ? "x" : "h", h, h.scalar_type(), h);
  if (c.residual) check_row_values("residual", *c.residual, h.scalar_type(), h);
  check_row_values("out_grad", c.out_grad, h.scalar_type(), h);
  if (c.sum_grad) check_row_values("h_grad", *c.sum_grad, h.scalar_type(), h);
  if (c.x_grad) check_row_values("x_grad", *c.x_grad, h.scalar_type(), h);
  if (c.residual_grad) check_row_values("residual_grad", *c.residual_grad, h.scalar_type(), h);
  TORCH_CHECK_VALUE(c.weight.scalar_type() == h.scalar_type() || c.weight.scalar_type() == at::kFloat, "weight must have dtype ", h.scalar_type(),
                    " or float32, got ", c.weight.scalar_type());
  a.weight = check_line("weight", c.weight, c.weight.scalar_type(), h.size(1), h);
  a.weight_dtype = layer_dtype(c.weight);
  a.rstd = static_cast<const float*>(check_line("rstd", c.rstd, at::kFloat, h.size(0), h));
  if (c.weight_grad) a.weight_grad = check_line("weight_grad", *c.weight_grad, c.weight.scalar_type(), h.size(1), h);
  if (drops(c.p)) a.rng_used = check_rng("rng_used", c.used, 2, h);
  if (h.size(1) == 0) return;
  a.out_grad = ptr(c.out_grad);
  a.out_grad_pitch = pitch(c.out_grad);
  (c.x ? a.x : a.sum) = ptr(h);
  (c.x ? a.x_pitch : a.sum_pitch) = pitch(h);
  if (c.residual) a.residual = ptr(*c.residual), a.residual_pitch = pitch(*c.residual);
  if (c.sum_grad) a.sum_grad = ptr(*c.sum_grad), a.sum_grad_pitch = pitch(*c.sum_grad);
  if (c.x_grad) a.x_grad = ptr(*c.x_grad), a.x_grad_pitch = pitch(*c.x_grad);
  if (c.residual_grad) a.residual_grad = ptr(*c.residual_grad), a.residual_grad_pitch = pitch(*c.residual_grad);
  a.rows = h.size(0);
  a.width = h.size(1);
  a.p = c.p;
  c10::cuda::CUDAGuard guard(h.device());
  Tensor ws;
  if (c.weight_grad) {
    a.workspace_bytes = fgms_b200_rms_norm_bwd_workspace_bytes(a.rows, a.width);
    if (a.workspace_bytes > 0) {
      ws = at::empty({(int64_t)a.workspace_bytes}, h.options().dtype(at::kByte).requires_grad(false));
      a.workspace = ws.data_ptr();
    }
  }
  check_status(fgms_b200_rms_norm_bwd(&a, stream_of(h)));
  for (const Tensor* t : {c.x_grad, c.residual_grad, c.weight_grad})
    if (t) written(*t);
}

void dropout(const Tensor& x, const Tensor& out, double p, const Tensor* rng, const Tensor* residual, const Tensor* used, bool backward) {
  fgms_b200_dropout_args a = {};
  a.dtype = layer_dtype(x);
  check_row_values(backward ? "out_grad" : "x", x, x.scalar_type(), x);
  check_row_values(backward ? "x_grad" : "out", out, x.scalar_type(), x);
  if (residual) check_row_values("residual", *residual, x.scalar_type(), x);
  if (!backward) a.rng = check_rng("rng", rng, 3, x);
  if (used || backward) a.rng_used = check_rng("rng_used", used, 2, x);
  if (x.size(1) == 0) return;
  a.x = ptr(x);
  a.x_pitch = pitch(x);
  a.out = ptr(out);
  a.out_pitch = pitch(out);
  if (residual) a.residual = ptr(*residual), a.residual_pitch = pitch(*residual);
  a.rows = x.size(0);
  a.width = x.size(1);
  a.p = p;
  c10::cuda::CUDAGuard guard(x.device());
  check_status(backward ? fgms_b200_dropout_bwd(&a, stream_of(x)) : fgms_b200_dropout(&a, stream_of(x)));
  written(out);
  if (!backward) written(*rng);
  if (!backward && used) written(*used);
}

// any shape as rows of its last dimension
Tensor as_rows(const Tensor& t) {
  if (t.dim() == 2 && t.is_contiguous()) return t;
  return (t.dim() == 0 ? t.reshape({1, 1}) : t.size(-1) == 0 ? t.reshape({0, 0}) : t.reshape({-1, t.size(-1)})).contiguous();
}
Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }
// a graph of the backward was asked for: it ends here, and says so to whoever goes through it
void end_graph(std::initializer_list<Tensor*> grads, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  for (Tensor* t : grads) {
    if (!t->defined()) continue;
    t->set_requires_grad(true);
    const auto ends = std::make_shared<torch::autograd::DelayedError>(what, 1);
    *t = (*ends)({*t})[0];
  }
}
const Tensor* maybe_tensor(const Tensor& t) { return t.defined() ? &t : nullptr; }

// Forward-mode differentiation is not built: a tangent would be dropped without a word where nothing needs a gradient.
void check_no_tangent(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode gradient");
}

void check_norm_shapes(const Tensor& x, const Tensor& weight, const Tensor* residual) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), "weight must have ", x.size(-1), " values, as many as a row");
  TORCH_CHECK_VALUE(!residual || residual->sizes() == x.sizes(), "residual must have the shape of x");
}

// Where the weight's gradient would see how the stored sum was rounded.
bool exact_sum_needed(const Tensor& x) { return x.scalar_type() != at::kFloat; }

// The norm of one call: out, and with a residual or dropout the sum that it is the norm of.
struct Normed {
  Tensor out, sum, rstd, used;  // 2-D, but out and sum
};
// `for_backward`: what a gradient needs is left as well; `from_x`: it will go by x and the residual instead of the sum
Normed norm_forward(const Tensor& x_, const Tensor& weight_, const Tensor* residual_, double eps, double p, const Tensor* rng, bool for_backward, bool from_x) {
  const Tensor x = as_rows(x_), weight = weight_.contiguous(), residual = residual_ ? as_rows(*residual_) : Tensor();
  Normed n;
  n.out = new_like(x_.is_contiguous() ? x_ : x);
  if (n.out.dim() != x_.dim()) n.out = n.out.view(x_.sizes());
  const bool drop = drops(p);
  const Tensor out = as_rows(n.out);
  Tensor sum;
  if (residual_ || (drop && for_backward && !from_x)) {
    n.sum = at::empty_like(n.out);
    sum = as_rows(n.sum);
  }
  if (for_backward) {
    n.rstd = at::empty({x.size(0)}, x.options().dtype(at::kFloat).requires_grad(false));
    if (drop) n.used = at::empty({2}, x.options().dtype(at::kLong).requires_grad(false));
  }
  rms_norm({x, &weight, out, maybe_tensor(residual), maybe_tensor(sum), nullptr, maybe_tensor(n.rstd), rng, maybe_tensor(n.used), eps, p});
  return n;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                                                const std::optional<Tensor>& residual, const std::optional<Tensor>& rng, double eps, double p) {
    const bool from_x = (residual || drops(p)) && weight.requires_grad() && exact_sum_needed(x);
    Normed n = norm_forward(x, weight, residual ? &*residual : nullptr, eps, p, rng ? &*rng : nullptr, true, from_x);
    ctx->saved_data["p"] = p;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["from_x"] = from_x;
    ctx->save_for_backward({from_x || !n.sum.defined() ? x : n.sum, weight, n.rstd, n.used, from_x && residual ? *residual : Tensor()});
    ctx->set_materialize_grads(false);
    if (residual) return {n.out, n.sum};
    return {n.out};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double p = ctx->saved_data["p"].toDouble();
    const bool residual = ctx->saved_data["residual"].toBool(), drop = drops(p);
    const Tensor h = as_rows(saved[0]), weight = saved[1].contiguous();
    const Tensor dy = grads[0].defined() ? as_rows(grads[0]) : at::zeros_like(h);
    const Tensor dsum = residual && grads[1].defined() ? as_rows(grads[1]) : Tensor();
    const bool want_x = ctx->needs_input_grad(0), want_residual = residual && ctx->needs_input_grad(2);
    Tensor x_grad, residual_grad, weight_grad;
    if (want_x) x_grad = new_like(h);
    if (want_residual && (drop || !want_x)) residual_grad = new_like(h);
    if (ctx->needs_input_grad(1)) weight_grad = new_like(weight);
    const bool from_x = ctx->saved_data["from_x"].toBool();
    const Tensor added = saved[4].defined() ? as_rows(saved[4]) : Tensor();
    rms_norm_bwd({dy, weight, saved[2], from_x ? nullptr : &h, from_x ? &h : nullptr, maybe_tensor(added), maybe_tensor(dsum), maybe_tensor(x_grad),
                  maybe_tensor(residual_grad), maybe_tensor(weight_grad), maybe_tensor(saved[3]), p});
    if (x_grad.defined()) x_grad = x_grad.view(saved[0].sizes());
    if (residual_grad.defined()) residual_grad = residual_grad.view(saved[0].sizes());
    if (want_residual && !residual_grad.defined()) residual_grad = x_grad;  // the same values
    if (at::GradMode::is_enabled() && residual_grad.defined() && residual_grad.is_same(x_grad)) residual_grad = x_grad.clone();
    end_graph({&x_grad, &weight_grad, &residual_grad}, "rms_norm is not differentiable twice");
    return {x_grad, weight_grad, residual_grad, Tensor(), Tensor(), Tensor()};
  }
};

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_, double p, const Tensor& rng, const std::optional<Tensor>& residual_) {
    const Tensor x = as_rows(x_), residual = residual_ ? as_rows(*residual_) : Tensor();
    const Tensor used = at::empty({2}, x.options().dtype(at::kLong).requires_grad(false)), out = new_like(x);
    dropout(x, out, p, &rng, maybe_tensor(residual), &used, false);
    ctx->saved_data["p"] = p;
    ctx->saved_data["residual"] = residual.defined();
    ctx->save_for_backward({used});
    return out.view(x_.sizes());
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor x_grad;
    if (ctx->needs_input_grad(0)) {
      const Tensor g = as_rows(grads[0]);
      x_grad = new_like(g);
      dropout(g, x_grad, ctx->saved_data["p"].toDouble(), nullptr, nullptr, &saved[0], true);
      x_grad = x_grad.view(grads[0].sizes());
      end_graph({&x_grad}, "dropout is not differentiable twice");
    }
    return {x_grad, Tensor(), Tensor(), ctx->saved_data["residual"].toBool() ? grads[0] : Tensor()};
  }
};

Tensor nn_dropout(const Tensor& x, double p, const Tensor& rng, const Tensor* residual) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK_VALUE(!residual || residual->sizes() == x.sizes(), "residual must have the shape of x");
  check_no_tangent("dropout", {&x, residual});
  if (at::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad())))
    return Dropout::apply(x, p, rng, residual ? std::optional<Tensor>(*residual) : std::nullopt);
  const Tensor rows = as_rows(x), other = residual ? as_rows(*residual) : Tensor(), out = new_like(rows);
  dropout(rows, out, p, &rng, maybe_tensor(other), nullptr, false);
  return out.view(x.sizes());
}

// Codes in rows that are multiples of 16 bytes apart, as the products in 8 bits like them.
Tensor new_codes(int64_t rows, int64_t width, const Tensor& like) {
  const auto options = like.options().dtype(at::kChar).requires_grad(false);
  const int64_t room = (width + 15) / 16 * 16;
  Tensor codes = at::empty({rows, room}, options);
  return room == width ? codes : codes.narrow(1, 0, width);
}
// (codes, scale, sum): without a weight there is no norm; the sum is undefined without a residual
std::array<Tensor, 3> rms_norm_int8(const Tensor& x_, const Tensor* weight_, const Tensor* residual_, double eps) {
  if (weight_) check_norm_shapes(x_, *weight_, residual_);
  check_no_tangent("an output in 8 bits", {&x_, weight_, residual_});
  TORCH_CHECK_VALUE(x_.dim() == 2, "x must have 2 dimensions, got ", x_.dim());
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && (x_.requires_grad() || (weight_ && weight_->requires_grad()) || (residual_ && residual_->requires_grad()))),
                    "codes of 8 bits have no gradient: call it under torch.no_grad()");
  const bool as_it_lies = (x_.stride(1) == 1 || x_.size(1) <= 1) && (x_.stride(0) >= x_.size(1) || x_.size(0) <= 1);
  const Tensor x = as_it_lies ? x_ : x_.contiguous(), weight = weight_ ? weight_->contiguous() : Tensor();
  const Tensor residual = residual_ ? as_rows(*residual_) : Tensor();
  std::array<Tensor, 3> r = {new_codes(x.size(0), x.size(1), x), at::empty({x.size(0)}, x.options().dtype(at::kFloat).requires_grad(false)),
                             residual_ ? at::empty({x.size(0), x.size(1)}, x.options().requires_grad(false)) : Tensor()};
  rms_norm({x, maybe_tensor(weight), r[0], maybe_tensor(residual), maybe_tensor(r[2]), &r[1], nullptr, nullptr, nullptr, eps, 0.0});
  return r;
}

// ---------------------------------------------------------------------------------------------
// products in 8 bits
// ---------------------------------------------------------------------------------------------
void grouped_i8(const Tensor& codes, const Tensor& scale, const Tensor& kernel, const Tensor& kernel_scale, const Tensor& out, const Tensor* kpos, bool zero_rest) {
  const int dtype = layer_dtype(out);
  TORCH_CHECK_VALUE(kernel.is_cuda() && kernel.scalar_type() == at::kChar && kernel.dim() == 3, "kernel must be an int8 CUDA tensor of 3 dimensions");
  const int64_t groups = kernel.size(0), c_out = kernel.size(1), c_in = kernel.size(2);
  TORCH_CHECK_VALUE(codes.device() == kernel.device(), "codes must live on ", kernel.device());
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar && codes.dim() == 2, "codes must be an int8 tensor of 2 dimensions");
  TORCH_CHECK_VALUE(codes.size(1) == c_in, "codes have ", codes.size(1), " channels, the kernel says ", c_in);
  TORCH_CHECK_VALUE(codes.numel() == 0 || c_in <= 1 || codes.stride(1) == 1, "codes must have the values of a row side by side");
  TORCH_CHECK_VALUE(codes.numel() == 0 || codes.size(0) <= 1 || codes.stride(0) >= c_in, "codes have rows that overlap");
  // the kernel's rows, of all groups alike
  const int64_t apart = c_out > 1 ? kernel.stride(1) : groups > 1 ? kernel.stride(0) : c_in;
  TORCH_CHECK_VALUE(kernel.numel() == 0 || ((c_in <= 1 || kernel.stride(2) == 1) && apart >= c_in && (groups <= 1 || c_out <= 1 || kernel.stride(0) == c_out * apart)),
                    "kernel must have the values of a row side by side, and all rows equally far apart");
  TORCH_CHECK_VALUE(scale.is_contiguous() && scale.dim() == 1 && scale.numel() == codes.size(0) && scale.scalar_type() == at::kFloat && scale.device() == kernel.device(),
                    "scale must be ", codes.size(0), " float32 values, one a row, on ", kernel.device());
  TORCH_CHECK_VALUE(kernel_scale.is_contiguous() && kernel_scale.dim() == 2 && kernel_scale.size(0) == groups && kernel_scale.size(1) == c_out &&
                        kernel_scale.scalar_type() == at::kFloat && kernel_scale.device() == kernel.device(),
                    "kernel_scale must be ", groups, " x ", c_out, " float32 values, one a channel, on ", kernel.device());
  check_feat("out", out, 2);
  TORCH_CHECK_VALUE(out.device() == kernel.device(), "out must live on ", kernel.device());
  TORCH_CHECK_VALUE(out.size(0) == codes.size(0) && out.size(1) == c_out, "out must be ", codes.size(0), " x ", c_out);
  if (kpos) {
    check_index("kpos", *kpos, kernel, 0);
    TORCH_CHECK_VALUE(kpos->dim() == 1 && kpos->size(0) == groups + 1, "kpos must have one entry more than there are groups: ", groups + 1, ", got ", kpos->numel());
  } else {
    TORCH_CHECK_VALUE(groups == 1, "kpos is needed for more than one group");
  }
  for (const int64_t n : {codes.size(0), c_in, c_out, groups}) TORCH_CHECK_VALUE(n <= 0x7fffffff, "more than 2^31 - 1 rows or channels");
  c10::cuda::CUDAGuard guard(kernel.device());
  const int8_t *a = static_cast<const int8_t*>(ptr(codes)), *b = static_cast<const int8_t*>(ptr(kernel));
  const int64_t a_pitch = pitch(codes);
  const int rows = (int)codes.size(0);
  const size_t bytes = fgms_b200_grouped_i8_workspace_bytes(a, a_pitch, b, apart, rows, (int)c_in, (int)c_out, (int)groups);
  const Tensor ws = bytes > 0 ? at::empty({(int64_t)bytes}, kernel.options().dtype(at::kByte).requires_grad(false)) : Tensor();
  check_status(fgms_b200_grouped_i8_fwd(a, a_pitch, static_cast<const float*>(ptr(scale)), b, apart, static_cast<const float*>(ptr(kernel_scale)), ptr(out),
                                        kpos ? iptr(*kpos) : nullptr, rows, (int)c_in, (int)c_out, (int)groups, dtype, zero_rest, space(ws), space_bytes(ws),
                                        stream_of(kernel)));
  written(out);
}

Tensor int8_linear(const Tensor& codes, const Tensor& scale, const Tensor& kernel_, const Tensor& kernel_scale_, const Tensor* kpos, at::ScalarType type) {
  const Tensor kernel = kernel_.dim() == 2 ? kernel_.unsqueeze(0) : kernel_, kernel_scale = kernel_scale_.dim() == 1 ? kernel_scale_.unsqueeze(0) : kernel_scale_;
  TORCH_CHECK_VALUE(kernel.is_cuda() && kernel.dim() == 3 && codes.dim() == 2, "kernel must be an int8 CUDA tensor of 2 or 3 dimensions, codes one of 2");
  check_no_tangent("int8_linear", {&scale, &kernel_scale_});
  Tensor out = at::empty({codes.size(0), kernel.size(1)}, kernel.options().dtype(type).requires_grad(false));
  grouped_i8(codes, scale, kernel, kernel_scale, out, kpos, kpos != nullptr);
  return out;
}

// ---------------------------------------------------------------------------------------------
// a layer of experts for a few tokens
// ---------------------------------------------------------------------------------------------
int activation_of(const std::string& name) {
  if (name == "silu") return FGMS_ACTIVATION_SILU;
  TORCH_CHECK_VALUE(name == "relu", "activation must be 'silu' or 'relu', got '", name, "'");
  return FGMS_ACTIVATION_RELU;
}

void expert_layer(const Tensor& x, const Tensor& router, const Tensor& w_in, const Tensor& w_out, const Tensor& out, const Tensor& experts, const Tensor& gates,
                  const std::string& activation) {
  check_no_tangent("expert_layer", {&x, &router, &w_in, &w_out});
  fgms_b200_expert_layer_args a = {};
  a.activation = activation_of(activation);
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2, "x must be a CUDA tensor of 2 dimensions");
  check_row_values("x", x, x.scalar_type(), x);
  a.dtype = layer_dtype(x);
  check_feat("w_in", w_in, 3, x);
  check_feat("w_out", w_out, 3, x);
  check_feat("router", router, 2);
  a.router_dtype = layer_dtype(router);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"w_in", w_in}, {"w_out", w_out}, {"router", router}, {"out", out}, {"experts", experts}, {"gates", gates}})
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " must live on ", x.device());
  const int64_t n = w_in.size(0), tokens = x.size(0), width = x.size(1), hidden = w_out.size(1), out_width = w_out.size(2), top_k = experts.dim() == 2 ? experts.size(1) : 0;
  TORCH_CHECK_VALUE(w_out.size(0) == n && router.size(0) == n, "w_in, w_out and router differ in experts");
  TORCH_CHECK_VALUE(w_in.size(1) == width && router.size(1) == width, "x has ", width, " channels, w_in ", w_in.size(1), ", the router ", router.size(1));
  a.gated = hidden > 0 && w_in.size(2) == 2 * hidden;
  TORCH_CHECK_VALUE(a.gated || w_in.size(2) == hidden, "w_in must be as wide as w_out is high, or twice that");
  TORCH_CHECK_VALUE(out.scalar_type() == x.scalar_type() && out.dim() == 2 && out.size(0) == tokens && out.size(1) == out_width &&
                        (out.numel() == 0 || out.stride(1) == 1) && (out.numel() == 0 || tokens <= 1 || out.stride(0) >= out_width),
                    "out must be ", tokens, " x ", out_width, " values of the rows' type, a row's side by side");
  TORCH_CHECK_VALUE(experts.scalar_type() == at::kInt && experts.dim() == 2 && experts.size(0) == tokens && experts.is_contiguous(),
                    "experts must be an int32 tensor of ", tokens, " x top_k");
  TORCH_CHECK_VALUE(gates.scalar_type() == at::kFloat && gates.sizes() == experts.sizes() && gates.is_contiguous(), "gates must be a float32 tensor of the shape of experts");
  for (const int64_t v : {n, tokens, width, hidden, out_width}) TORCH_CHECK_VALUE(v <= 0x7fffffff, "more than 2^31 - 1 rows or channels");
  a.x = ptr(x);
  a.router = ptr(router);
  a.w_in = ptr(w_in);
  a.w_out = ptr(w_out);
  a.out = ptr(out);
  a.chosen = static_cast<int32_t*>(ptr(experts));
  a.gates = static_cast<float*>(ptr(gates));
  a.x_pitch = pitch(x);
  a.out_pitch = pitch(out);
  a.tokens = (int)tokens;
  a.experts = (int)n;
  a.top_k = (int)top_k;
  a.width = (int)width;
  a.hidden = (int)hidden;
  a.out_width = (int)out_width;
  c10::cuda::CUDAGuard guard(x.device());
  a.workspace_bytes = fgms_b200_expert_layer_workspace_bytes(a.tokens, a.experts, a.top_k, a.hidden, a.out_width);
  const Tensor ws = a.workspace_bytes > 0 ? at::empty({(int64_t)a.workspace_bytes}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
  a.workspace = space(ws);
  check_status(fgms_b200_expert_layer(&a, stream_of(x)));
  for (const Tensor* t : {&out, &experts, &gates}) written(*t);
}

// ---------------------------------------------------------------------------------------------
// AdamW over many tensors
// ---------------------------------------------------------------------------------------------
int adamw_dtype(const char* name, const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return FGMS_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return FGMS_DTYPE_BF16;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "unsupported ", name, " dtype ", t.scalar_type(), ": float16, bfloat16 or float32");
  return FGMS_DTYPE_F32;
}

// The tensors of the caller's lists, which hold them for the length of the call: a hundred references counted up and down cost as much as the launch.
using TensorList = std::vector<const Tensor*>;
struct AdamwLists {
  TensorList params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_scales, exp_avg_sq_scales;  // masters: null where there is none
};

void adamw(const AdamwLists& a, const Tensor& step, const Tensor& lr_tensor, const Tensor& grad_scale, const Tensor& found_inf, fgms_b200_adamw_options o) {
  const size_t n = a.params.size();
  TORCH_CHECK_VALUE(step.is_cuda() && step.scalar_type() == at::kInt && step.numel() == 2 && step.is_contiguous(),
                    "step must be a contiguous int32 CUDA tensor of two entries: the steps done, and 0");
  const auto device = step.device();
  auto one = [&](const char* name, const Tensor& t) -> const float* {
    if (!t.defined()) return nullptr;
    TORCH_CHECK_VALUE(t.device() == device && t.scalar_type() == at::kFloat && t.numel() == 1, name, " must be one float32 value on ", device);
    return t.data_ptr<float>();
  };
  o.lr_device = one("lr", lr_tensor);
  o.grad_scale = one("grad_scale", grad_scale);
  o.found_inf = one("found_inf", found_inf);
  o.step = step.data_ptr<int32_t>();
  const bool eight = !a.exp_avg_scales.empty() || !a.exp_avg_sq_scales.empty() || (n > 0 && a.exp_avgs.size() == n && a.exp_avgs[0]->scalar_type() == at::kFloat8_e4m3fn);
  o.state_bits = eight ? 8 : 32;
  auto length = [&](const char* name, size_t got) { TORCH_CHECK_VALUE(got == n, name, " has ", got, " tensors, params ", n); };
  length("grads", a.grads.size());
  length("exp_avgs", a.exp_avgs.size());
  length("exp_avg_sqs", a.exp_avg_sqs.size());
  if (!a.masters.empty()) length("masters", a.masters.size());
  if (eight) {
    length("exp_avg_scales", a.exp_avg_scales.size());
    length("exp_avg_sq_scales", a.exp_avg_sq_scales.size());
  }
  std::vector<fgms_b200_adamw_tensor> list(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = *a.params[i], &g = *a.grads[i], &m = *a.exp_avgs[i], &v = *a.exp_avg_sqs[i];
    auto check = [&](const char* name, const Tensor& t, int64_t count, at::ScalarType type) {
      TORCH_CHECK_VALUE(t.device() == device, name, " ", i, " must live on ", device, ", got ", t.device());
      TORCH_CHECK_VALUE(t.is_contiguous(), name, " ", i, " must be contiguous");
      TORCH_CHECK_VALUE(t.numel() == count, name, " ", i, " must have ", count, " values, got ", t.numel());
      TORCH_CHECK_VALUE(t.scalar_type() == type, name, " ", i, " must have dtype ", type, ", got ", t.scalar_type());
    };
    const int64_t count = p.numel(), blocks = (count + 127) / 128;
    const at::ScalarType moment = eight ? at::kFloat8_e4m3fn : at::kFloat;
    check("param", p, count, p.scalar_type());
    check("grad", g, count, g.scalar_type());
    check("exp_avg", m, count, moment);
    check("exp_avg_sq", v, count, moment);
    fgms_b200_adamw_tensor& t = list[i];
    t = {};
    t.count = count;
    t.param = ptr(p);
    t.grad = ptr(g);
    t.exp_avg = ptr(m);
    t.exp_avg_sq = ptr(v);
    t.param_dtype = adamw_dtype("parameter", p);
    t.grad_dtype = adamw_dtype("gradient", g);
    if (!a.masters.empty() && a.masters[i]) {
      check("master", *a.masters[i], count, at::kFloat);
      t.master = static_cast<float*>(ptr(*a.masters[i]));
    }
    if (eight) {
      check("exp_avg_scale", *a.exp_avg_scales[i], blocks, at::kFloat);
      check("exp_avg_sq_scale", *a.exp_avg_sq_scales[i], blocks, at::kFloat);
      t.exp_avg_scale = static_cast<float*>(ptr(*a.exp_avg_scales[i]));
      t.exp_avg_sq_scale = static_cast<float*>(ptr(*a.exp_avg_sq_scales[i]));
    }
  }
  c10::cuda::CUDAGuard guard(device);
  check_status(fgms_b200_adamw(list.data(), (int)n, &o, stream_of(step)));
  written(step);
  for (const auto* tensors : {&a.params, &a.exp_avgs, &a.exp_avg_sqs, &a.masters, &a.exp_avg_scales, &a.exp_avg_sq_scales})
    for (const Tensor* t : *tensors)
      if (t) written(*t);
}

// ---------------------------------------------------------------------------------------------
// Python entry points (positional arguments only; the functions of backend.py / nn.py give them their names)
// ---------------------------------------------------------------------------------------------
const Tensor& feat_arg(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
const Tensor& index_arg(PyObject* o, const char* name) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), name, " must be an int32 tensor");
  return THPVariable_Unpack(o);
}
const Tensor* optional_arg(PyObject* o, const char* name) { return o == Py_None ? nullptr : &index_arg(o, name); }
int64_t int_arg(PyObject* o) {  // like int(o): a Python or NumPy integer, or a tensor of one element
  PyObject* n = PyLong_CheckExact(o) ? Py_NewRef(o) : PyNumber_Long(o);
  if (!n) throw python_error();
  const long long v = PyLong_AsLongLong(n);
  Py_DECREF(n);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void expect(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got); }

PyObject* py_fusion_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const Tensor &in_feats = feat_arg(a[0], "in_feats"), &kernel = feat_arg(a[1], "kernel"), &out = feat_arg(a[3], "out_feats");
  const Tensor &kpos = index_arg(a[4], "kpos"), *qkpos = optional_arg(a[5], "qkpos");
  const Tensor &in_map = index_arg(a[6], "in_map"), &out_map = index_arg(a[7], "out_map");
  fusion_fwd(in_feats, kernel, int_arg(a[2]), out, kpos, qkpos, in_map, out_map, bool_arg(a[8]), bool_arg(a[9]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_seq_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const Tensor &in_feats = feat_arg(a[0], "in_feats"), &kernel = feat_arg(a[1], "kernel"), &out = feat_arg(a[3], "out_feats");
  const Tensor &nnz = index_arg(a[4], "kernel_nnz"), &kpos = index_arg(a[5], "kpos");
  const Tensor &in_map = index_arg(a[6], "in_map"), &out_map = index_arg(a[7], "out_map");
  seq_fwd(in_feats, kernel, int_arg(a[2]), out, nnz, kpos, in_map, out_map, bool_arg(a[8]), bool_arg(a[9]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 13);
  const Tensor &grad_out = feat_arg(a[0], "out_feats_grad"), &in_feats = feat_arg(a[1], "in_feats"), &kernel = feat_arg(a[2], "kernel");
  const Tensor &in_grad = feat_arg(a[4], "in_feats_grad"), &kernel_grad = feat_arg(a[5], "kernel_grad");
  const Tensor &kpos = index_arg(a[6], "kpos"), *qkpos = optional_arg(a[7], "qkpos");
  const Tensor &in_map = index_arg(a[8], "in_map"), &out_map = index_arg(a[9], "out_map");
  bwd(grad_out, in_feats, kernel, int_arg(a[3]), in_grad, kernel_grad, kpos, qkpos, in_map, out_map, bool_arg(a[10]), bool_arg(a[11]),
      bool_arg(a[12]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_sparse_conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  const Tensor &feats = feat_arg(a[0], "in_feats"), &weight = feat_arg(a[1], "kernel");
  const Tensor &kpos = index_arg(a[2], "kpos"), &imap = index_arg(a[3], "in_map"), &omap = index_arg(a[4], "out_map");
  return THPVariable_Wrap(SparseConv::apply(feats, weight, kpos, imap, omap, int_arg(a[5]), bool_arg(a[6])));
  END_HANDLE_TH_ERRORS
}
std::vector<const Tensor*> tensor_list(PyObject* list, const char* name, bool gaps = false) {
  TORCH_CHECK_TYPE(PyList_Check(list) || PyTuple_Check(list), name, " must be a list of tensors");
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  std::vector<const Tensor*> out;
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(list, i);
    out.push_back(gaps && o == Py_None ? nullptr : &feat_arg(o, name));
  }
  return out;
}
double double_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

// (params, grads, exp_avgs, exp_avg_sqs, step, lr, beta1, beta2, eps, weight_decay, masters, exp_avg_scales, exp_avg_sq_scales, seed, grad_scale, found_inf)
PyObject* py_adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 16);
  AdamwLists lists;
  lists.params = tensor_list(a[0], "params");
  lists.grads = tensor_list(a[1], "grads");
  lists.exp_avgs = tensor_list(a[2], "exp_avgs");
  lists.exp_avg_sqs = tensor_list(a[3], "exp_avg_sqs");
  if (a[10] != Py_None) lists.masters = tensor_list(a[10], "masters", true);
  if (a[11] != Py_None) lists.exp_avg_scales = tensor_list(a[11], "exp_avg_scales");
  if (a[12] != Py_None) lists.exp_avg_sq_scales = tensor_list(a[12], "exp_avg_sq_scales");
  fgms_b200_adamw_options o = {};
  Tensor lr_tensor;
  if (THPVariable_Check(a[5])) lr_tensor = THPVariable_Unpack(a[5]);
  if (lr_tensor.defined() && !lr_tensor.is_cuda()) {
    TORCH_CHECK_VALUE(lr_tensor.numel() == 1, "lr must be one value");
    o.lr = lr_tensor.item<double>();
    lr_tensor = Tensor();
  } else if (!lr_tensor.defined()) {
    o.lr = double_arg(a[5]);
  }
  o.beta1 = double_arg(a[6]);
  o.beta2 = double_arg(a[7]);
  o.eps = double_arg(a[8]);
  o.weight_decay = double_arg(a[9]);
  const int64_t seed = int_arg(a[13]);
  TORCH_CHECK_VALUE(seed >= 0 && seed <= 0xffffffffll, "seed must be in [0, 2^32)");
  o.seed = (uint32_t)seed;
  auto maybe = [](PyObject* t, const char* name) { return t == Py_None ? Tensor() : feat_arg(t, name); };
  adamw(lists, feat_arg(a[4], "step"), lr_tensor, maybe(a[14], "grad_scale"), maybe(a[15], "found_inf"), o);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (in_feats, [kernels], [kpos, in_map, out_map of every map], [src, skip, map, n_in, n_out of every layer], arch80) -> the last layer's
// output, or None where the layers are to be run one by one
PyObject* py_sparse_stack(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  const Tensor& feats = feat_arg(a[0], "in_feats");
  auto tensors = [](PyObject* list, const char* name) {
    TORCH_CHECK_TYPE(PyList_Check(list), name, " must be a list");
    std::vector<Tensor> out;
    out.reserve(PyList_GET_SIZE(list));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) out.push_back(feat_arg(PyList_GET_ITEM(list, i), name));
    return out;
  };
  const std::vector<Tensor> weights = tensors(a[1], "kernels"), maps = tensors(a[2], "maps");
  TORCH_CHECK_TYPE(PyList_Check(a[3]), "plan must be a list");
  StackPlan plan;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[3]); ++i) plan.push_back(int_arg(PyList_GET_ITEM(a[3], i)));
  const bool arch80 = bool_arg(a[4]);
  if (!stack_suits(feats, weights, maps, plan, arch80)) Py_RETURN_NONE;
  return THPVariable_Wrap(SparseStack::apply(feats, at::TensorList(weights), at::TensorList(maps), plan, arch80));
  END_HANDLE_TH_ERRORS
}
PyObject* py_wgrad_fp32_sums(PyObject*, PyObject* const* a, Py_ssize_t n) {  // () -> the switch; (value) sets it
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n <= 1, "expected at most 1 argument, got ", n);
  if (n == 1) g_fp32_sums.store(bool_arg(a[0]), std::memory_order_relaxed);
  return PyBool_FromLong(g_fp32_sums.load(std::memory_order_relaxed));
  END_HANDLE_TH_ERRORS
}
PyObject* py_fwd_os(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  const Tensor &in_feats = feat_arg(a[0], "in_feats"), &kernel = feat_arg(a[1], "kernel"), &out = feat_arg(a[2], "out_feats");
  const Tensor &nbr = index_arg(a[3], "nbr"), *bias = a[5] == Py_None ? nullptr : &feat_arg(a[5], "bias");
  fwd_os(in_feats, kernel, out, nbr, bool_arg(a[4]), bias, bool_arg(a[6]), bool_arg(a[7]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_grouped_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  grouped_fwd(feat_arg(a[0], "in_feats"), feat_arg(a[1], "kernel"), feat_arg(a[2], "out_feats"), index_arg(a[3], "kpos"), bool_arg(a[4]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_grouped_dgrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  grouped_dgrad(feat_arg(a[0], "out_feats_grad"), feat_arg(a[1], "kernel"), feat_arg(a[2], "in_feats_grad"), index_arg(a[3], "kpos"), bool_arg(a[4]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_grouped_wgrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  grouped_wgrad(feat_arg(a[0], "in_feats"), feat_arg(a[1], "out_feats_grad"), feat_arg(a[2], "kernel_grad"), index_arg(a[3], "kpos"));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_grouped_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  return THPVariable_Wrap(GroupedLinear::apply(feat_arg(a[0], "feats"), feat_arg(a[1], "weight"), index_arg(a[2], "kpos")));
  END_HANDLE_TH_ERRORS
}

// (voxels per level, [(kpos, imap, omap) ...], [coords of level 1 ...]), or None for a cloud that does not suit
PyObject* py_build_pyramid(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const Pyramid r = build_pyramid(index_arg(a[0], "coords"), (int)int_arg(a[1]), (int)int_arg(a[2]));
  if (!r.fits) Py_RETURN_NONE;
  PyObject *voxels = PyList_New(r.voxels.size()), *maps = PyList_New(r.maps.size()), *coords = PyList_New(r.out_coords.size());
  for (size_t i = 0; i < r.voxels.size(); ++i) PyList_SET_ITEM(voxels, i, PyLong_FromLongLong(r.voxels[i]));
  for (size_t i = 0; i < r.maps.size(); ++i) {
    PyObject* t = PyTuple_New(3);
    for (int k = 0; k < 3; ++k) PyTuple_SET_ITEM(t, k, THPVariable_Wrap(r.maps[i][k]));
    PyList_SET_ITEM(maps, i, t);
  }
  for (size_t i = 0; i < r.out_coords.size(); ++i) PyList_SET_ITEM(coords, i, THPVariable_Wrap(r.out_coords[i]));
  return Py_BuildValue("(NNN)", voxels, maps, coords);
  END_HANDLE_TH_ERRORS
}

const Tensor* maybe_arg(PyObject* o, const char* name) { return o == Py_None ? nullptr : &feat_arg(o, name); }

// (x, weight, out, eps, residual, residual_out, scale, rstd, p, rng, rng_used)
PyObject* py_rms_norm_into(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 11);
  rms_norm({feat_arg(a[0], "x"), &feat_arg(a[1], "weight"), feat_arg(a[2], "out"), maybe_arg(a[4], "residual"), maybe_arg(a[5], "residual_out"),
            maybe_arg(a[6], "scale"), maybe_arg(a[7], "rstd"), maybe_arg(a[9], "rng"), maybe_arg(a[10], "rng_used"), double_arg(a[3]), double_arg(a[8])});
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (out_grad, h, weight, rstd, x_grad, weight_grad, h_grad, residual_grad, p, rng_used, x, residual)
PyObject* py_rms_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 12);
  rms_norm_bwd({feat_arg(a[0], "out_grad"), feat_arg(a[2], "weight"), feat_arg(a[3], "rstd"), maybe_arg(a[1], "h"), maybe_arg(a[10], "x"),
                maybe_arg(a[11], "residual"), maybe_arg(a[6], "h_grad"), maybe_arg(a[4], "x_grad"), maybe_arg(a[7], "residual_grad"), maybe_arg(a[5], "weight_grad"), maybe_arg(a[9], "rng_used"), double_arg(a[8])});
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (x, out, p, rng, residual, rng_used)
PyObject* py_dropout_into(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  dropout(feat_arg(a[0], "x"), feat_arg(a[1], "out"), double_arg(a[2]), &feat_arg(a[3], "rng"), maybe_arg(a[4], "residual"), maybe_arg(a[5], "rng_used"), false);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (out_grad, x_grad, p, rng_used)
PyObject* py_dropout_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  dropout(feat_arg(a[0], "out_grad"), feat_arg(a[1], "x_grad"), double_arg(a[2]), nullptr, nullptr, &feat_arg(a[3], "rng_used"), true);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (x, codes, scale)
PyObject* py_quantize_rows_into(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const Tensor& scale = feat_arg(a[2], "scale");
  rms_norm({feat_arg(a[0], "x"), nullptr, feat_arg(a[1], "codes"), nullptr, nullptr, &scale, nullptr, nullptr, nullptr, 0.0, 0.0});
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (x, weight, eps, residual, p, rng): out, or with a residual (out, sum)
PyObject* py_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const Tensor &x = feat_arg(a[0], "x"), &weight = feat_arg(a[1], "weight"), *residual = maybe_arg(a[3], "residual"), *rng = maybe_arg(a[5], "rng");
  const double eps = double_arg(a[2]), p = double_arg(a[4]);
  check_norm_shapes(x, weight, residual);
  check_no_tangent("rms_norm", {&x, &weight, residual});
  Tensor out, sum;
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()))) {
    auto r = RmsNorm::apply(x, weight, residual ? std::optional<Tensor>(*residual) : std::nullopt, rng ? std::optional<Tensor>(*rng) : std::nullopt, eps, p);
    out = r[0];
    if (residual) sum = r[1];
  } else {
    const Normed r = norm_forward(x, weight, residual, eps, p, rng, false, false);
    out = r.out;
    sum = r.sum;
  }
  if (!residual) return THPVariable_Wrap(out);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(sum));
  END_HANDLE_TH_ERRORS
}
// (x, weight or None, eps, residual): (codes, scale), or with a residual (codes, scale, sum)
PyObject* py_rms_norm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const Tensor* residual = maybe_arg(a[3], "residual");
  const auto r = rms_norm_int8(feat_arg(a[0], "x"), maybe_arg(a[1], "weight"), residual, double_arg(a[2]));
  if (!residual) return Py_BuildValue("(NN)", THPVariable_Wrap(r[0]), THPVariable_Wrap(r[1]));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(r[0]), THPVariable_Wrap(r[1]), THPVariable_Wrap(r[2]));
  END_HANDLE_TH_ERRORS
}
// (x, p, rng, residual)
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  return THPVariable_Wrap(nn_dropout(feat_arg(a[0], "x"), double_arg(a[1]), feat_arg(a[2], "rng"), maybe_arg(a[3], "residual")));
  END_HANDLE_TH_ERRORS
}

// (codes, scale, kernel, kernel_scale, out, kpos, zero_rest)
PyObject* py_grouped_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  grouped_i8(feat_arg(a[0], "codes"), feat_arg(a[1], "scale"), feat_arg(a[2], "kernel"), feat_arg(a[3], "kernel_scale"), feat_arg(a[4], "out"),
             optional_arg(a[5], "kpos"), bool_arg(a[6]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (codes, scale, kernel, kernel_scale, kpos, dtype)
PyObject* py_int8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  TORCH_CHECK_TYPE(THPDtype_Check(a[5]), "dtype must be a torch.dtype");
  return THPVariable_Wrap(int8_linear(feat_arg(a[0], "codes"), feat_arg(a[1], "scale"), feat_arg(a[2], "kernel"), feat_arg(a[3], "kernel_scale"),
                                      optional_arg(a[4], "kpos"), reinterpret_cast<THPDtype*>(a[5])->scalar_type));
  END_HANDLE_TH_ERRORS
}

// (x, router, w_in, w_out, out, experts, gates, activation)
PyObject* py_expert_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  TORCH_CHECK_TYPE(PyUnicode_Check(a[7]), "activation must be a string");
  const char* activation = PyUnicode_AsUTF8(a[7]);
  if (!activation) throw python_error();
  expert_layer(feat_arg(a[0], "x"), feat_arg(a[1], "router"), feat_arg(a[2], "w_in"), feat_arg(a[3], "w_out"), feat_arg(a[4], "out"), feat_arg(a[5], "experts"),
               feat_arg(a[6], "gates"), activation);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FGMS_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FGMS_METHOD("fusion_fwd", py_fusion_fwd), FGMS_METHOD("seq_fwd", py_seq_fwd),         FGMS_METHOD("bwd", py_bwd),
    FGMS_METHOD("fwd_os", py_fwd_os),         FGMS_METHOD("sparse_conv", py_sparse_conv),
    FGMS_METHOD("sparse_stack", py_sparse_stack),
    FGMS_METHOD("wgrad_fp32_sums", py_wgrad_fp32_sums),
    FGMS_METHOD("grouped_fwd", py_grouped_fwd), FGMS_METHOD("grouped_dgrad", py_grouped_dgrad),
    FGMS_METHOD("grouped_wgrad", py_grouped_wgrad), FGMS_METHOD("grouped_linear", py_grouped_linear),
    FGMS_METHOD("adamw", py_adamw),
    FGMS_METHOD("rms_norm_into", py_rms_norm_into), FGMS_METHOD("rms_norm_bwd", py_rms_norm_bwd), FGMS_METHOD("rms_norm", py_rms_norm),
    FGMS_METHOD("rms_norm_int8", py_rms_norm_int8), FGMS_METHOD("quantize_rows_into", py_quantize_rows_into),
    FGMS_METHOD("dropout_into", py_dropout_into), FGMS_METHOD("dropout_bwd", py_dropout_bwd), FGMS_METHOD("dropout", py_dropout),
    FGMS_METHOD("grouped_i8", py_grouped_i8), FGMS_METHOD("int8_linear", py_int8_linear),
    FGMS_METHOD("expert_layer", py_expert_layer),
    FGMS_METHOD("build_pyramid", py_build_pyramid), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module_def); }
