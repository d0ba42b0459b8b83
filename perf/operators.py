"""Products of ragged groups of rows with a weight matrix each, and the AdamW update of many tensors at once: as cases that can be
timed and whose outputs can be compared.

With ``own`` true a pass makes the calls that a user makes (``backend.fgms_grouped_*_cuda``, ``nn.grouped_linear``,
``backend.fgms_adamw_cuda``); otherwise it computes the same from elementary torch operations.

``kind`` says what a pass is:

* ``forward``      rows ``kpos[g] .. kpos[g + 1]`` of the features times matrix ``g``; rows of no group stay as they were
* ``input_grad``   the same rows of the output gradient times the transposed matrix ``g``
* ``weight_grad``  the gradient of every matrix: features transposed times output gradient over the rows of its group
* ``train``        all three through ``nn.grouped_linear`` and autograd; rows of no group are zero
* ``adamw``        one step over all tensors, moments in 32 bits, or in 8 (e4m3 with a scale for each 128 values, rounded up or
                   down at random so that the mean is kept)

``rows`` are the rows of all groups together, ``rest`` those behind the last group; ``spread`` is how unevenly the rows fall to the
groups (0: evenly; from about 1 on some groups are many times as large as others, and some are empty), ``split`` the seed of that.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ELEM = {"fp16": 2, "bf16": 2, "fp32": 4}
PRODUCTS = ("forward", "input_grad", "weight_grad", "train")
BLOCK = 128         # values that share a scale
E4M3_MAX = 448.0
SMALLEST = 2.0 ** -100  # a block whose largest value is below this is held as zeros
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
GRAD_SCALE = 1024.0
STEPS_DONE, SEED = 10, 7


def _product(name, kind, dtype, rows, groups, c_in, c_out, spread=0.5, rest=0, split=1):
    c = {"kind": kind, "dtype": dtype, "rows": rows, "groups": groups, "c_in": c_in, "c_out": c_out, "spread": spread, "rest": rest, "split": split}
    return {**c, "name": name} if name else c


def _adamw(name, dtype, master, bits, layers, values, split=1):
    """``layers``: ``unet`` for the 25 layers of the encoder-decoder stack, or ``drawn`` for as many tensors as ``tensors``
    of ragged sizes, about ``values`` in all."""
    c = {"kind": "adamw", "dtype": dtype, "master": master, "bits": bits, "tensors": layers, "values": values, "split": split}
    return {**c, "name": name} if name else c


def listed():
    return [
        # serving, one token: the two groups it goes to, all latency
        _product("forward_one_token", "forward", "bf16", 2, 8, 512, 512, spread=0.0),
        # serving, a batch of single tokens over many groups: every weight is read for a row or two
        _product("forward_tokens", "forward", "bf16", 96, 64, 2048, 1024, spread=0.7, rest=32),
        # a middle-sized ragged batch, widths that no tile divides, rows behind the last group
        _product("forward_ragged", "forward", "fp16", 5003, 12, 1000, 1496, spread=0.8, rest=57),
        # fp32 storage and arithmetic
        _product("forward_fp32", "forward", "fp32", 6007, 9, 260, 516, spread=0.6),
        # a long prompt, or a training batch's forward
        _product("forward_large", "forward", "bf16", 32768, 32, 2048, 4096, spread=0.3),
        # the two halves of a backward by themselves
        _product("input_grad", "input_grad", "bf16", 16384, 16, 2048, 2048, spread=0.4),
        _product("weight_grad", "weight_grad", "fp16", 16411, 16, 2048, 1024, spread=0.6, rest=101),
        # a training step of a layer through autograd
        _product("train_layer", "train", "bf16", 8192, 8, 1024, 4096, spread=0.3),
        # the encoder-decoder's weights after a backward in fp16 with a loss scale, fp32 masters
        _adamw("adamw_unet", "fp16", True, 32, 25, 0),
        # a larger network in fp32
        _adamw("adamw_fp32_large", "fp32", False, 32, 48, 150_000_000),
        # a small head in bf16 without masters, moments in 8 bits, sizes that no block divides
        _adamw("adamw8_bf16_small", "bf16", False, 8, 17, 900_000),
        # a larger network in fp16 with masters, moments in 8 bits
        _adamw("adamw8_fp16_large", "fp16", True, 8, 61, 120_000_000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, odd):
    w = _log(rng, lo, hi)
    return w if odd else max(8, w // 8 * 8)


def draw(rng):
    split = rng.randrange(1 << 30)
    if rng.random() < 0.3:
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        return _adamw(None, dtype, dtype != "fp32" and rng.random() < 0.6, rng.choice([32, 8]), _log(rng, 1, 100), _log(rng, 1000, 100_000_000), split)
    kind = rng.choice(["forward", "forward", "input_grad", "weight_grad", "train"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp16", "fp32"])
    odd = rng.random() < 0.2  # widths whose rows are not multiples of 16 bytes
    most = 1024 if odd or dtype == "fp32" else 4096
    a, b = _width(rng, 64, most, odd), _width(rng, 64, most, odd)
    groups = _log(rng, 1, 64)
    while groups * a * b > 1 << 28:
        groups //= 2
    budget = (3e9 if odd or dtype == "fp32" else 2.5e11) / (3 if kind == "train" else 1)
    rows = _log(rng, 1, max(2, min(32768, int(budget / (2.0 * a * b)))))
    return _product(None, kind, dtype, rows, groups, a, b, round(rng.uniform(0, 1), 2), rng.choice([0, 0, rng.randrange(1, 200)]), split)


def sizes(case):
    """Rows of every group: ``rows`` shared out in proportion to weights that are log-normal, the remainder at random."""
    rng = random.Random(case["split"])
    share = [math.exp(rng.gauss(0, 1) * case["spread"]) for _ in range(case["groups"])]
    total = sum(share)
    n = [int(case["rows"] * s / total) for s in share]
    for _ in range(case["rows"] - sum(n)):
        n[rng.choices(range(case["groups"]), weights=share)[0]] += 1
    return n


def counts(case):
    """Values of every tensor of an update."""
    if case["values"] == 0:
        widths = [4, 32, 32, 64, 128, 256]
        pair = [(widths[s], widths[s + 1]) for s in range(1, 5)]
        down = [n for a, b in pair for n in (8 * a * b, 27 * b * b, 27 * b * b)]
        up = [n for a, b in reversed(pair) for n in (8 * a * b, 27 * a * a, 27 * a * a)]
        return [27 * widths[0] * widths[1]] + down + up
    rng = random.Random(case["split"])
    share = [math.exp(rng.gauss(0, 1.2)) for _ in range(case["tensors"])]
    return [max(1, int(case["values"] * s / sum(share))) for s in share]


def _placed(case):
    """Where every tensor lies in a buffer of all of them, from a multiple of 128 values: ([(first, count)], total)."""
    at, placed = 0, []
    for n in counts(case):
        placed.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return placed, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["kind"] == "adamw":
        placed, total = _placed(case)
        dtype = DTYPE[case["dtype"]]
        real = torch.zeros(total, device="cuda")
        for at, n in placed:
            real[at:at + n] = 1.0
        size = torch.exp(normal(total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-3  # gradients of rows differ in size
        grad = normal(total) * size * real
        scaled = case["dtype"] == "fp16"
        s = {"kind": "adamw", "bits": case["bits"], "placed": placed, "real": real, "param": (normal(total) * 0.02 * real).to(dtype),
             "grad": (grad * (GRAD_SCALE if scaled else 1.0)).to(dtype),
             "grad_scale": torch.full((1,), GRAD_SCALE, device="cuda") if scaled else None,
             "step": torch.tensor([STEPS_DONE, 0], dtype=torch.int32, device="cuda")}
        if case["master"]:
            s["master"] = s["param"].float() + normal(total) * 1e-6 * real
        m, v = normal(total) * size * 0.3 * real, (normal(total) * size).square() * 0.01 * real
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
        else:
            for name, x in (("m", m), ("v", v)):
                s[name + "_scale"] = x.view(-1, BLOCK).abs().amax(1) / E4M3_MAX
                s[name] = (x.view(-1, BLOCK) / s[name + "_scale"].clamp(min=1e-30)[:, None]).clamp(-E4M3_MAX, E4M3_MAX).view(-1).to(torch.float8_e4m3fn)
        lists = {k: [s[k][at:at + n] for at, n in placed] for k in ("param", "grad", "master", "m", "v") if k in s}
        lists |= {k: [s[k][at // BLOCK:(at + n + BLOCK - 1) // BLOCK] for at, n in placed] for k in ("m_scale", "v_scale") if k in s}
        s["lists"] = lists
        return s
    dtype, n = DTYPE[case["dtype"]], sizes(case)
    kpos = [0]
    for k in n:
        kpos.append(kpos[-1] + k)
    rows = case["rows"] + case["rest"]
    a, b, kind = case["c_in"], case["c_out"], case["kind"]

    def features(width):
        x = normal(rows, width)
        x[case["rows"]:] = math.nan  # whatever a buffer with room to spare holds behind its rows
        return x.to(dtype)

    s = {"kind": kind, "kpos": torch.tensor(kpos, dtype=torch.int32, device="cuda"), "most": max(n), "groups": case["groups"]}
    if kind != "weight_grad":
        s["weight"] = ((torch.rand((case["groups"], a, b), generator=gen, device="cuda") * 2 - 1) * a ** -0.5).to(dtype)
    if kind != "input_grad":
        s["feats"] = features(a)
    if kind != "forward":
        s["grad"] = features(b)
    if kind == "forward":
        s["out"] = torch.full((rows, b), 0.5, dtype=dtype, device="cuda")
    if kind == "input_grad":
        s["feats_grad"] = torch.full((rows, a), 0.5, dtype=dtype, device="cuda")
    if kind == "weight_grad":
        s["weight_grad"] = torch.full((case["groups"], a, b), 0.5, dtype=dtype, device="cuda")
    if kind == "train":
        s["feats"].requires_grad_()
        s["weight"].requires_grad_()
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _places(s, rows):
    """Rows of every group side by side: [groups, most], and which of them there are; the others are row ``rows``."""
    at = s["kpos"][:-1, None] + torch.arange(s["most"], device="cuda")
    there = at < s["kpos"][1:, None]
    return torch.where(there, at, rows), there


def _gathered(x, at, there):
    return torch.where(there[..., None], x[at.clamp(max=x.size(0) - 1)].float(), 0.0)


def _scattered(y, at, into):
    """``into`` with the rows of the groups in their places (and one row more, for the places of no row)."""
    full = torch.cat([into, into[:1]])
    full[at] = y.to(into.dtype)
    return full[:-1]


def _plain_product(s):
    kind = s["kind"]
    rows = s["feats" if kind != "input_grad" else "grad"].size(0)
    at, there = _places(s, rows)
    x = _gathered(s["feats"].detach(), at, there) if "feats" in s else None
    g = _gathered(s["grad"], at, there) if "grad" in s else None
    w = s["weight"].detach().float() if "weight" in s else None
    if kind == "forward":
        return _scattered(torch.bmm(x, w), at, s["out"])
    if kind == "input_grad":
        return _scattered(torch.bmm(g, w.transpose(1, 2)), at, s["feats_grad"])
    if kind == "weight_grad":
        return torch.bmm(x.transpose(1, 2), g).to(s["feats"].dtype)
    return {"out": _scattered(torch.bmm(x, w), at, torch.zeros_like(s["grad"])),
            "feats_grad": _scattered(torch.bmm(g, w.transpose(1, 2)), at, torch.zeros_like(s["feats"].detach())),
            "weight_grad": torch.bmm(x.transpose(1, 2), g).to(s["feats"].dtype)}


def _mix(h):
    """The finalizer of MurmurHash3 on 32-bit numbers (held in 64 bits)."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _e4m3(x, lot, floor):
    """``x`` in e4m3 with a scale for each 128 values, rounded up with the probability of the part that would be cut off: ``lot`` is
    uniform in 0 .. 65535.  ``floor``: what is above zero stays above it."""
    n = x.numel()
    room = (n + BLOCK - 1) // BLOCK * BLOCK
    x = torch.nn.functional.pad(x, (0, room - n)).view(-1, BLOCK)
    lot = torch.nn.functional.pad(lot, (0, room - n)).view(-1, BLOCK).int()
    largest = x.abs().amax(1, keepdim=True)
    held = largest >= SMALLEST
    scale = torch.where(held, largest * (1.0 / E4M3_MAX), 0.0)
    u = torch.where(held, x.abs() * torch.where(held, torch.ones_like(scale) / scale, 0.0), 0.0).clamp(max=E4M3_MAX)
    normal = ((u.view(torch.int32) + (lot << 4)) & -(1 << 20)).view(torch.float32)
    small = torch.floor(u * 512.0 + lot.float() * (1.0 / 65536.0))
    if floor:
        small = torch.where(u > 0, small.clamp(min=1.0), small)
    code = torch.copysign(torch.where(u >= 2.0 ** -6, normal, small * (1.0 / 512.0)), x)
    return code.view(-1)[:n].to(torch.float8_e4m3fn), scale.view(-1)


def _held(code, scale):
    n = code.numel()
    return code.float() * scale.repeat_interleave(BLOCK)[:n]


def _plain_update(s, i, now, key):
    p, g, m, v = (s["lists"][k][i] for k in ("param", "grad", "m", "v"))
    t = now.double()
    rate, root = (LR / (1.0 - BETA1 ** t)).float(), (1.0 / torch.sqrt(1.0 - BETA2 ** t)).float()
    master = s["lists"]["master"][i] if "master" in s else None
    g = g.float()
    if s["grad_scale"] is not None:
        g = g * (torch.ones_like(s["grad_scale"]) / s["grad_scale"])
    if s["bits"] == 8:
        m, v = _held(m, s["lists"]["m_scale"][i]), _held(v, s["lists"]["v_scale"][i])
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    w = p.float() if master is None else master
    w = w * (1.0 - LR * DECAY) - rate * (m / (torch.sqrt(v) * root + EPS))
    if s["bits"] == 8:
        h = _mix((torch.arange(p.numel(), device="cuda") * 0x9E3779B1 + key) & 0xFFFFFFFF)
        for name, x, lot in (("m", m, h & 0xFFFF), ("v", v, h >> 16)):
            code, scale = _e4m3(x, lot, floor=name == "v")
            s["lists"][name][i].copy_(code)
            s["lists"][name + "_scale"][i].copy_(scale)
    else:
        s["lists"]["m"][i].copy_(m)
        s["lists"]["v"][i].copy_(v)
    if master is not None:
        master.copy_(w)
    p.copy_(w)


def _plain_adamw(s):
    now = s["step"][0] + 1
    key = _mix((now.long() * 0x9E3779B9 & 0xFFFFFFFF) ^ SEED)
    [_plain_update(s, i, now, key) for i in range(len(s["placed"]))]
    s["step"][0] += 1


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if kind == "adamw":
        if own:
            from fgms_b200 import backend
            lists = s["lists"]
            backend.fgms_adamw_cuda(lists["param"], lists["grad"], lists["m"], lists["v"], s["step"], LR, BETA1, BETA2, EPS, DECAY,
                                    masters=lists.get("master"), exp_avg_scales=lists.get("m_scale"), exp_avg_sq_scales=lists.get("v_scale"),
                                    seed=SEED, grad_scale=s["grad_scale"])
        else:
            _plain_adamw(s)
        return {k: s[k] for k in ("param", "master", "m", "v", "m_scale", "v_scale", "step") if k in s}
    if own:
        from fgms_b200 import backend, nn
        if kind == "forward":
            backend.fgms_grouped_fwd_cuda(s["feats"], s["weight"], s["out"], s["kpos"])
            return s["out"]
        if kind == "input_grad":
            backend.fgms_grouped_dgrad_cuda(s["grad"], s["weight"], s["feats_grad"], s["kpos"])
            return s["feats_grad"]
        if kind == "weight_grad":
            backend.fgms_grouped_wgrad_cuda(s["feats"], s["grad"], s["weight_grad"], s["kpos"])
            return s["weight_grad"]
        out = nn.grouped_linear(s["feats"], s["weight"], s["kpos"])
        feats_grad, weight_grad = torch.autograd.grad(out, (s["feats"], s["weight"]), s["grad"])
        return {"out": out.detach(), "feats_grad": feats_grad, "weight_grad": weight_grad}
    return _plain_product(s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "adamw":
        n, e = float(sum(counts(case))), ELEM[case["dtype"]]
        weights = e + 8 if case["master"] else 2 * e  # with a master the parameter itself is written only
        moments = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
        return {"bytes": n * (weights + e + moments), "flops": 15.0 * n}
    n, a, b, e = sizes(case), case["c_in"], case["c_out"], ELEM[case["dtype"]]
    rows, used = float(sum(n)), float(sum(k > 0 for k in n))
    flops = 2.0 * rows * a * b
    if case["kind"] in ("forward", "input_grad"):
        return {"bytes": e * (rows * (a + b) + used * a * b), "flops": flops}
    if case["kind"] == "weight_grad":
        return {"bytes": e * (rows * (a + b) + case["groups"] * float(a * b)), "flops": flops}
    return {"bytes": e * (2 * rows * (a + b) + (used + case["groups"]) * a * b), "flops": 3 * flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adamw":
        t = STEPS_DONE + 1
        g = s["grad"].double()
        if s["grad_scale"] is not None:
            g /= GRAD_SCALE
        m, v = s["m"].double(), s["v"].double()
        if case["bits"] == 8:
            m *= s["m_scale"].double().repeat_interleave(BLOCK)
            v *= s["v_scale"].double().repeat_interleave(BLOCK)
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        w = s["master"].double() if case["master"] else s["param"].double()
        w = (1 - LR * DECAY) * w - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out = {"param": w, "step": None}
        if case["master"]:
            out["master"] = w
        if case["bits"] == 32:
            return {**out, "m": m, "v": v}
        return {**out, "m": None, "v": None, "m_scale": v.new_tensor(m.view(-1, BLOCK).abs().amax(1) / E4M3_MAX),
                "v_scale": v.new_tensor(v.view(-1, BLOCK).amax(1) / E4M3_MAX)}
    n, at = sizes(case), 0
    first = []
    for k in n:
        first.append(at)
        at += k
    take = lambda x, g: x[first[g]:first[g] + n[g]].double()
    weight, kind = s.get("weight"), case["kind"]

    def rows_of(x, like, transposed, blank):
        out = torch.full((x.size(0), like), blank, dtype=torch.float64, device="cuda")
        for g in range(len(n)):
            w = weight[g].detach().double()
            out[first[g]:first[g] + n[g]] = take(x, g) @ (w.T if transposed else w)
        return out

    def weights_of():
        return torch.stack([take(s["feats"].detach(), g).T @ take(s["grad"], g) for g in range(len(n))])

    if kind == "forward":
        return rows_of(s["feats"], case["c_out"], False, 0.5)
    if kind == "input_grad":
        return rows_of(s["grad"], case["c_in"], True, 0.5)
    if kind == "weight_grad":
        return weights_of()
    return {"out": rows_of(s["feats"].detach(), case["c_out"], False, 0.0), "feats_grad": rows_of(s["grad"], case["c_in"], True, 0.0),
            "weight_grad": weights_of()}
