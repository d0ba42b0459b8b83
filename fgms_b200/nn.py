"""Autograd wrapper around the operator: what dgSPARSE-Lib (the caller named by the reference's README)
puts on top of ``FGMS.backend``.

``sparse_conv(feats, weight, kmap)`` is differentiable in ``feats`` and ``weight``; forward is
``fgms_fusion_fwd_cuda``, backward is ``fgms_bwd_cuda`` (dgrad + wgrad).  ``SparseConv3d`` is the
``nn.Module`` that owns the ``[k_vol, c_in, c_out]`` weight.  Kernel maps are passed in (a
:class:`fgms_b200.gpu_maps.DeviceKernelMap`, or anything with ``kpos / imap / omap / n_in / n_out``
device tensors): layers at one resolution share one map, which is the map caching the reference's driver
does by loading one file per layer shape (``spconv-test.py:63-73``).
"""
from __future__ import annotations

import math

import torch

from . import _native, backend

__all__ = ["sparse_conv", "sparse_conv_inference", "SparseConv3d", "SparseUNet", "grouped_linear", "GroupedLinear", "rms_norm", "RMSNorm",
           "rms_norm_int8", "quantize_rows", "rng_state", "recomputed", "dropout", "Dropout", "int8_linear", "Int8GroupedLinear", "expert_layer", "ExpertLayer"]


def sparse_conv(feats: torch.Tensor, weight: torch.Tensor, kmap, arch80: bool = True) -> torch.Tensor:
    """``out[omap[j]] += feats[imap[j]] @ weight[k(j)]`` over the pairs of ``kmap``; differentiable."""
    if feats.size(0) != kmap.n_in:
        raise ValueError(f"feats has {feats.size(0)} rows, the kernel map expects {kmap.n_in}")
    if weight.size(0) != kmap.kpos.numel() - 1:
        raise ValueError("weight and kernel map disagree on the number of offsets")
    return _native.sparse_conv(feats, weight, kmap.kpos, kmap.imap, kmap.omap, kmap.n_out, arch80)


def sparse_conv_inference(feats: torch.Tensor, weight: torch.Tensor, kmap, bias: torch.Tensor | None = None,
                          relu: bool = False, arch80: bool = True) -> torch.Tensor:
    """Forward only, through the output-stationary kernel (``backend.fgms_fwd_os_cuda``): every output row is
    written once — the same bits on every run — with ``bias`` and ReLU applied in the kernel's epilogue (a
    batch-norm layer in inference form is a scaled weight and a bias).  No autograd.  The neighbour table the
    kernel reads is built on first use and kept on ``kmap``.  Tensor-core shapes only (fp16, or fp32 storage
    with tf32 arithmetic; channel counts multiples of 16 up to 256)."""
    if feats.size(0) != kmap.n_in:
        raise ValueError(f"feats has {feats.size(0)} rows, the kernel map expects {kmap.n_in}")
    nbr = getattr(kmap, "_neighbor_table", None)
    if nbr is None:
        nbr = backend.build_neighbor_table(kmap.kpos, kmap.imap, kmap.omap, kmap.n_in, kmap.n_out)
        try:
            kmap._neighbor_table = nbr
        except AttributeError:  # a map type without room for it: rebuilt on every call
            pass
    out = torch.empty((kmap.n_out, weight.size(2)), dtype=feats.dtype, device=feats.device)
    with torch.no_grad():
        backend.fgms_fwd_os_cuda(feats.contiguous(), weight.detach().contiguous(), out, nbr, arch80, bias=bias, relu=relu)
    return out


class SparseConv3d(torch.nn.Module):
    """Sparse 3-D convolution layer with a ``[k_vol, c_in, c_out]`` weight (no bias, like the reference's
    operator); initialised like ``torch.nn.Conv3d`` (kaiming uniform, a = sqrt(5), fan_in = c_in * k_vol)."""

    def __init__(self, c_in: int, c_out: int, k_vol: int = 27, dtype=torch.float16, device="cuda", arch80: bool = True):
        super().__init__()
        self.c_in, self.c_out, self.k_vol, self.arch80 = c_in, c_out, k_vol, arch80
        bound = 1.0 / math.sqrt(c_in * k_vol)
        w = (torch.rand((k_vol, c_in, c_out), device=device, dtype=torch.float32) * 2 - 1) * bound
        self.weight = torch.nn.Parameter(w.to(dtype))

    def forward(self, feats: torch.Tensor, kmap) -> torch.Tensor:
        return sparse_conv(feats, self.weight, kmap, self.arch80)


def grouped_linear(feats: torch.Tensor, weight: torch.Tensor, kpos: torch.Tensor) -> torch.Tensor:
    """``out[r] = feats[r] @ weight[g]`` for the rows ``kpos[g] <= r < kpos[g + 1]`` of every group; differentiable in ``feats`` and
    ``weight``.  Rows of no group (a buffer with room to spare) are zero in the output and in the gradient of ``feats``, whatever they
    hold.  Rows in the order of their groups come from a stable sort by group: ``order = ids.argsort(stable=True)``,
    ``kpos = torch.searchsorted(ids[order], torch.arange(groups + 1, device=...), out_int32=True)``."""
    return _native.grouped_linear(feats, weight, kpos)


class GroupedLinear(torch.nn.Module):
    """One ``c_in -> c_out`` matrix for each of ``groups`` groups of rows (experts), a ``[groups, c_in, c_out]`` weight initialised like
    ``torch.nn.Linear``; ``forward(feats, kpos)`` is :func:`grouped_linear`."""

    def __init__(self, c_in: int, c_out: int, groups: int, dtype=torch.float16, device="cuda"):
        super().__init__()
        self.c_in, self.c_out, self.groups = c_in, c_out, groups
        bound = 1.0 / math.sqrt(c_in)
        w = (torch.rand((groups, c_in, c_out), device=device, dtype=torch.float32) * 2 - 1) * bound
        self.weight = torch.nn.Parameter(w.to(dtype))

    def forward(self, feats: torch.Tensor, kpos: torch.Tensor) -> torch.Tensor:
        return grouped_linear(feats, self.weight, kpos)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None, dropout: float = 0.0,
             rng: torch.Tensor | None = None):
    """``h * weight / sqrt(mean(h ** 2) + eps)`` over the last dimension of ``h = residual + dropout(x)``; differentiable in ``x``, ``weight`` and
    ``residual``.  With a ``residual`` the result is ``(out, h)``, ``h`` being what the next layer adds to; without one it is ``out``.  One pass over
    the rows for all of it.  ``weight`` is of the type of ``x`` or float32.  ``rng``: see :func:`dropout`; a call that drops nothing (``dropout = 0``) leaves it alone."""
    return _native.rms_norm(x, weight, eps, residual, dropout, rng)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """:func:`rms_norm` with the output in 8 bits, for the products behind it: ``(codes, scale)`` or ``(codes, scale, h)``, where
    ``codes * scale[:, None]`` is the normed row.  ``x`` has two dimensions.  Codes are int8 rows that start 16 bytes apart.  No autograd."""
    return _native.rms_norm_int8(x, weight, eps, residual)


def quantize_rows(x: torch.Tensor):
    """``(codes, scale)``: the rows of ``x``, which has two dimensions and up to 32768 columns, in 8 bits with a float32 scale each.  No autograd."""
    return _native.rms_norm_int8(x, None, 0.0, None)


def int8_linear(codes: torch.Tensor, scale: torch.Tensor, kernel: torch.Tensor, kernel_scale: torch.Tensor, kpos: torch.Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(codes * scale[:, None]) @ (kernel * kernel_scale[:, None]).T`` in 8-bit integers, exact up to the scales, in ``dtype``: ``codes`` from
    :func:`rms_norm_int8` or :func:`quantize_rows`, ``kernel`` ``[c_out, c_in]`` with a scale a channel, or ``[groups, c_out, c_in]`` with ``kpos`` as in
    :func:`grouped_linear` (rows of no group are zero).  No autograd."""
    return _native.int8_linear(codes, scale, kernel, kernel_scale, kpos, dtype)


def _spaced(kernel: torch.Tensor) -> torch.Tensor:
    """The codes ``[groups, c_out, c_in]`` with a channel's a multiple of 16 bytes from the next one's, as the products read them: a copy that made them dense (a move to another
    device) would have every call copy all of them first."""
    groups, c_out, c_in = kernel.shape
    room = (c_in + 15) // 16 * 16
    if kernel.stride() == (c_out * room, room, 1) and (kernel.is_meta or kernel.data_ptr() % 16 == 0):
        return kernel
    spaced = torch.zeros((groups, c_out, room), dtype=kernel.dtype, device=kernel.device)[:, :, :c_in]
    return spaced.copy_(kernel)


class Int8GroupedLinear(torch.nn.Module):
    """:class:`GroupedLinear` for serving: its matrices in 8 bits with a scale for each channel, rows in 8 bits with a scale each.
    ``forward(feats, kpos)`` takes rows, or the ``(codes, scale)`` of :func:`rms_norm_int8` and :func:`quantize_rows`; the output is of ``dtype``, or
    the type that ``weight`` had.  A cast of the module (``.bfloat16()``) changes neither that nor the scales, which stay float32.  At most 32768
    channels in, as many as :func:`quantize_rows` takes."""

    def __init__(self, weight: torch.Tensor, dtype: torch.dtype | None = None):
        super().__init__()
        groups, c_in, c_out = weight.shape
        codes, scale = quantize_rows(weight.detach().transpose(1, 2).reshape(groups * c_out, c_in))
        self.register_buffer("kernel", _spaced(codes.as_strided((groups, c_out, c_in), (c_out * codes.stride(0), codes.stride(0), 1))))
        self.register_buffer("kernel_scale", scale.view(groups, c_out))
        self.dtype = weight.dtype if dtype is None else dtype

    def _apply(self, fn, recurse=True):
        scale = self.kernel_scale
        super()._apply(fn, recurse)
        if self.kernel_scale.dtype != torch.float32:  # whatever a model's rows and weights are cast to
            self.kernel_scale = scale.to(self.kernel_scale.device)
        self.kernel = _spaced(self.kernel)
        return self

    def _load_from_state_dict(self, *args):
        super()._load_from_state_dict(*args)
        self.kernel = _spaced(self.kernel)

    def __setstate__(self, state):
        super().__setstate__(state)
        self.kernel = _spaced(self.kernel)

    def forward(self, feats, kpos: torch.Tensor | None = None) -> torch.Tensor:
        codes, scale = feats if isinstance(feats, tuple) else quantize_rows(feats)
        return int8_linear(codes, scale, self.kernel, self.kernel_scale, kpos, self.dtype)


def rng_state(seed: int = 0, device="cuda") -> torch.Tensor:
    """The state of :func:`dropout`'s generator on a device: ``[seed, calls made, 0]``."""
    if not 0 <= seed < 2 ** 63:
        raise ValueError("seed must be in [0, 2^63)")
    return torch.tensor([seed, 0, 0], dtype=torch.int64, device=device)


class _From:
    """While it is open, the states go on from where ``first`` says they were; without ``again`` it notes that."""

    def __init__(self, states, first, again):
        self.states, self.first, self.again, self.later = states, first, again, None

    def __enter__(self):
        was = [s.clone() for s in self.states]
        if not self.again:
            self.first[:] = was
            return
        self.later = was
        for s, f in zip(self.states, self.first):
            s.copy_(f)

    def __exit__(self, *_):
        if self.again:
            for s, now in zip(self.states, self.later):
                s.copy_(now)


def recomputed(*of):
    """What ``torch.utils.checkpoint`` needs for a segment that drops values, as its ``context_fn``::

        checkpoint(block, x, use_reentrant=False, context_fn=lambda: nn.recomputed(block))

    A segment that is computed again for its backward would count its calls again and drop other values than the ones that made the loss, so that its gradients would belong
    to another mask.  With this it goes by the calls of the first time, and the states are left as they were.  ``of``: states (:func:`rng_state`), and modules whose
    :class:`Dropout` and :class:`RMSNorm` layers are meant.  Copies on the device alone: it can be captured into a graph (with ``preserve_rng_state=False``)."""
    states = []
    for o in of:
        found = [m.rng for m in o.modules() if isinstance(m, (Dropout, RMSNorm)) and m.rng is not None] if isinstance(o, torch.nn.Module) else [o]
        states += [s for s in found if not any(s is t for t in states)]
    if not all(isinstance(s, torch.Tensor) and s.dtype == torch.int64 and s.shape == (3,) for s in states):
        raise ValueError("states of rng_state, or modules, are needed")
    first = []
    return _From(states, first, False), _From(states, first, True)


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + x * kept / (1 - p)``, with a mask that is never stored: the backward draws the same lots again.  ``rng`` comes from
    :func:`rng_state` and counts the calls, on the device: a replayed graph drops other values every time.  Differentiable in ``x`` and
    ``residual``.  The lots of a value hang on its row and column, the last dimension being the columns.  A call with ``p = 0`` counts too.  Segments that are computed again
    for their backward (``torch.utils.checkpoint``) need :func:`recomputed`."""
    return _native.dropout(x, p, rng, residual)


def _module_state(seed: int | None, device) -> torch.Tensor:
    """The state of a module's generator.  Lots hang on (seed, call, row, column) alone: modules of one seed drop the same values in every step.  Without a seed it is
    drawn from PyTorch's generator of the host (``torch.manual_seed`` repeats it), moved apart by the rank where there are several."""
    if seed is None:
        seed = int(torch.randint(2 ** 63 - 1, (), dtype=torch.int64, device="cpu"))
        if torch.distributed.is_available() and torch.distributed.is_initialized():
            seed = (seed + torch.distributed.get_rank() * 0x9E3779B97F4A7C15) % 2 ** 63  # an odd number: no two ranks alike
    return rng_state(seed, device)


class RMSNorm(torch.nn.Module):
    """:func:`rms_norm` with its weight; ``forward(x)`` is the normed rows, ``forward(x, residual)`` those and the sum.  ``dropout`` is applied to ``x`` in
    training, with a state of its own, the buffer ``rng``; ``seed``: see :class:`Dropout`."""

    def __init__(self, width: int, eps: float = 1e-6, dropout: float = 0.0, dtype=torch.float32, device="cuda", seed: int | None = None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout must be in [0, 1], got {dropout}")
        self.width, self.eps, self.dropout = width, eps, dropout
        self.weight = torch.nn.Parameter(torch.ones(width, dtype=dtype, device=device))
        self.register_buffer("rng", _module_state(seed, device) if dropout > 0 else None)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        p = self.dropout if self.training else 0.0
        return rms_norm(x, self.weight, self.eps, residual, p, self.rng)


class Dropout(torch.nn.Module):
    """:func:`dropout` with a state of its own, the buffer ``rng``; outside training ``x``, or ``residual + x``.

    ``seed``: None draws another one for every module, from PyTorch's generator of the host, and every rank of an initialised process group has its own.
    Modules of one seed, copies of a module and ranks whose buffers are one rank's (a checkpoint, ``broadcast_buffers`` of
    ``DistributedDataParallel``) drop the same values: ``module.rng.copy_(rng_state(another))`` moves them apart."""

    def __init__(self, p: float = 0.5, device="cuda", seed: int | None = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        self.p = p
        self.register_buffer("rng", _module_state(seed, device))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if self.training and self.p > 0:
            return dropout(x, self.p, self.rng, residual)
        return x if residual is None else residual + x


_FEW_TOKENS, _MOST_EXPERTS, _MOST_CHOSEN = 64, 512, 16  # what backend.fgms_expert_layer_cuda takes


def _few_tokens(x, router, w_in, w_out, top_k) -> bool:
    needs_grad = torch.is_grad_enabled() and any(t.requires_grad for t in (x, router, w_in, w_out))
    return (not needs_grad and 0 < x.size(0) <= _FEW_TOKENS and router.size(0) <= _MOST_EXPERTS and top_k <= _MOST_CHOSEN
            and x.dtype in (torch.float16, torch.bfloat16) and w_in.dtype == w_out.dtype == x.dtype and router.dtype in (x.dtype, torch.float32)
            and x.size(1) % 8 == 0 and w_out.size(1) % 8 == 0 and w_out.size(2) % 8 == 0
            and all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (x, router, w_in, w_out)))


def _library_has_32_bits() -> bool:
    """Whether a library product of float32 matrices is one: a process may allow TF32, which keeps 10 bits of the operands, or be inside autocast, which keeps fewer."""
    try:
        return not torch.backends.cuda.matmul.allow_tf32 and not torch.is_autocast_enabled("cuda")
    except RuntimeError:  # it was allowed under another name
        return False


def _logits(rows, router):
    """``rows @ router.T`` in 32 bits: a choice hangs on the difference of two.  By the library where it has them (16384 rows of 4096 to 64 experts 353 us, 840 with
    gradients), otherwise by the grouped products, as one group (443 and 1170)."""
    n = rows.size(0)
    if n == 0 or _library_has_32_bits():
        return rows.float() @ router.float().T
    return grouped_linear(rows.float(), router.float().T[None], torch.arange(0, n + 1, n, dtype=torch.int32, device=rows.device))


def expert_layer(x: torch.Tensor, router: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, top_k: int, activation: str = "silu") -> torch.Tensor:
    """Each row of ``x`` through the ``top_k`` of its experts that the ``router`` (``[experts, width]``) gives the largest logits, their outputs added up with
    the softmax over those as weights.  An expert is ``h @ w_out[e]`` with ``h = act(x @ w_in[e])``, or ``act(u[:, :hidden]) * u[:, hidden:]`` where
    ``w_in`` is twice as wide as ``w_out`` is high; ``activation`` is ``"silu"`` or ``"relu"``.

    Up to 64 rows of float16 or bfloat16 that need no gradient take two launches (:func:`fgms_b200.backend.fgms_expert_layer_cuda`; it chooses by logits in
    64 bits, the other way by logits in 32, whatever the process allows library products; a logit that is not a number is the lowest in
    both).  Otherwise rows are put in the order of their experts and go through :func:`grouped_linear`:
    differentiable in ``x``, ``router`` (through the weights of the sum), ``w_in`` and ``w_out``."""
    if activation not in ("silu", "relu"):
        raise ValueError(f"activation must be 'silu' or 'relu', got {activation!r}")
    experts, hidden = w_in.size(0), w_out.size(1)
    if router.dim() != 2 or router.size(0) != experts or w_out.size(0) != experts or not 1 <= top_k <= experts:
        raise ValueError(f"router, w_in and w_out must have the same experts, and at least top_k = {top_k} of them")
    if w_in.size(2) not in (hidden, 2 * hidden):
        raise ValueError("w_in must be as wide as w_out is high, or twice that")
    rows = x.reshape(-1, x.size(-1))
    if _few_tokens(rows, router, w_in, w_out, top_k):
        out = torch.empty((rows.size(0), w_out.size(2)), dtype=x.dtype, device=x.device)
        chosen = torch.empty((rows.size(0), top_k), dtype=torch.int32, device=x.device)
        with torch.no_grad():
            backend.fgms_expert_layer_cuda(rows, router, w_in, w_out, out, chosen, torch.empty(chosen.shape, device=x.device), activation)
        return out.view(*x.shape[:-1], w_out.size(2))
    logits = _logits(rows, router)
    logits = torch.where(logits != logits, float("-inf"), logits)  # a sort would put what is not a number first
    value, chosen = (t[:, :top_k] for t in torch.sort(logits, dim=1, descending=True, stable=True))
    gate = torch.softmax(value, 1)
    ids = chosen.reshape(-1)
    order = ids.argsort(stable=True)
    kpos = torch.searchsorted(ids[order], torch.arange(experts + 1, device=x.device), out_int32=True)
    u = grouped_linear(rows[order // top_k], w_in, kpos)
    act = torch.nn.functional.silu if activation == "silu" else torch.relu
    h = act(u[:, :hidden]) * u[:, hidden:] if u.size(1) == 2 * hidden and hidden else act(u)
    y = grouped_linear(h, w_out, kpos)
    back = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=x.device))
    out = (y[back].float().view(rows.size(0), top_k, w_out.size(2)) * gate[:, :, None]).sum(1)
    return out.to(x.dtype).view(*x.shape[:-1], w_out.size(2))


class ExpertLayer(torch.nn.Module):
    """A layer of ``experts`` experts of ``hidden`` channels, of which every row takes ``top_k``: :func:`expert_layer` with its weights, initialised
    like ``torch.nn.Linear``.  ``gated``: ``w_in`` is twice as wide, ``act(first half) * second half``."""

    def __init__(self, width: int, hidden: int, experts: int, top_k: int, gated: bool = True, activation: str = "silu", dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        if not 1 <= top_k <= experts:
            raise ValueError(f"top_k must be in [1, {experts}], got {top_k}")
        self.top_k, self.activation = top_k, activation
        made = lambda fan_in, *shape: torch.nn.Parameter(((torch.rand(shape, device=device) * 2 - 1) / math.sqrt(fan_in)).to(dtype))
        self.router = made(width, experts, width)
        self.w_in = made(width, experts, width, (2 if gated else 1) * hidden)
        self.w_out = made(hidden, experts, hidden, width)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return expert_layer(x, self.router, self.w_in, self.w_out, self.top_k, self.activation)


_LAYER_FORWARD = SparseConv3d.forward
_MODULE = torch.nn.modules.module
_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _watched() -> bool:
    """Whether something beyond the layers themselves sees or transforms their calls.  PyTorch answers most of this under private names
    only: a release that lacks one counts as watching.  Several ranks count too, because gradients that leave with their layer are
    exchanged beside the rest of the backward."""
    try:
        return (torch._C._get_tracing_state() is not None or torch.compiler.is_compiling() or torch.autograd.forward_ad._current_level >= 0
                or torch._C._functorch.peek_interpreter_stack() is not None
                or torch._C._autograd._top_saved_tensors_default_hooks(True) is not None
                or torch._C._len_torch_dispatch_stack() > 0 or torch._C._len_torch_function_stack() > 0
                or (torch.distributed.is_available() and torch.distributed.is_initialized())
                or bool(_MODULE._global_forward_hooks or _MODULE._global_forward_pre_hooks
                        or _MODULE._global_backward_hooks or _MODULE._global_backward_pre_hooks))
    except AttributeError:
        return True


def _one_node(layers) -> bool:
    """Whether a stack may run as one autograd node: nothing sees the calls of its layers."""
    if _watched() or SparseConv3d.forward is not _LAYER_FORWARD or SparseConv3d.__call__ is not torch.nn.Module.__call__:
        return False
    for layer in layers:
        d = layer.__dict__
        if type(layer) is not SparseConv3d or "forward" in d or d["arch80"] != layers[0].__dict__["arch80"] or any(d.get(h, True) for h in _HOOKS):
            return False
    return True


class SparseUNet(torch.nn.Module):
    """The encoder-decoder stack of :mod:`fgms_b200.unet` as an ``nn.Module`` over the autograd operator: one
    :class:`SparseConv3d` per layer of the specification, decoder skips added to the transposed convolutions'
    outputs.  ``forward(feats, umaps)`` takes the kernel maps of all resolutions (``unet.build_unet_maps``)."""

    def __init__(self, spec, dtype=torch.float16, device="cuda", arch80: bool = True):
        super().__init__()
        self.spec = list(spec)
        self.layers = torch.nn.ModuleList(
            SparseConv3d(l.c_in, l.c_out, l.k_vol, dtype=dtype, device=device, arch80=arch80) for l in self.spec)

    def load_weights(self, weights):
        with torch.no_grad():
            for layer, w in zip(self.layers, weights):
                layer.weight.copy_(torch.as_tensor(w).to(layer.weight.device, layer.weight.dtype))

    def _forward_as_one(self, feats: torch.Tensor, umaps):
        """The stack as one autograd node (``csrc/torch_binding.cpp``), or None: see :func:`_one_node`."""
        layers = list(self.layers)
        if not layers or len(layers) != len(self.spec) or type(feats) is not torch.Tensor or not _one_node(layers):
            return None
        value, seen, weights, maps, plan = {"input": 0}, {}, [], [], []
        for spec, layer in zip(self.spec, layers):
            w, km = layer._parameters.get("weight"), umaps.of(spec)
            if type(w) is not torch.nn.Parameter or spec.src not in value or (spec.skip is not None and spec.skip not in value):
                return None
            m, _ = seen.setdefault(id(km), (len(seen), km))  # with the map itself: an id is one object's for as long as it lives
            if 3 * m == len(maps):
                maps += km.kpos, km.imap, km.omap
            plan += value[spec.src], -1 if spec.skip is None else value[spec.skip], m, km.n_in, km.n_out
            weights.append(w)
            value[spec.dst] = len(weights)
        if not all(type(t) is torch.Tensor for t in maps):
            return None
        return _native.sparse_stack(feats, weights, maps, plan, layers[0].arch80)

    def forward(self, feats: torch.Tensor, umaps) -> torch.Tensor:
        out = self._forward_as_one(feats, umaps)
        if out is not None:
            return out
        val = {"input": feats}
        for spec, layer in zip(self.spec, self.layers):
            y = layer(val[spec.src], umaps.of(spec))
            if spec.skip is not None:
                y = y + val[spec.skip]
            val[spec.dst] = y
        return val[self.spec[-1].dst]
