"""What stands between two layers of experts, and such a layer in its serving forms, as cases that can be timed and whose outputs can be
compared: the root-mean-square norm with the residual's addition, dropout whose mask is never stored, products of 8-bit integers with scales, and
a whole layer of experts for a few tokens.

With ``own`` true a pass makes the calls that a user makes (``nn.rms_norm``, ``nn.rms_norm_int8``, ``nn.int8_linear``, ``nn.dropout``,
``backend.fgms_grouped_i8_fwd_cuda``, ``backend.fgms_expert_layer_cuda``); otherwise it computes the same from elementary torch operations.

``kind`` says what a pass is:

* ``norm``          rows plus their residual, normed; the sum is an output too
* ``norm_train``    the same with dropout on the rows, and the gradients of rows, residual and weight
* ``norm8_linear``  rows plus their residual, normed into 8 bits with a scale a row, times a matrix in 8 bits with a scale a channel
* ``linear8``       rows in 8 bits of ragged groups times a matrix in 8 bits each; rows of no group stay as they were
* ``dropout``       residual plus what dropout leaves of the rows, and with ``train`` the gradient of the rows
* ``experts``       router, choice of ``top_k`` experts for each token, first product, activation, second product, weighted sum

Dropout's lots are 16 bits each of Philox 4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): key the seed, counter
(column / 8, row, number of the call); a value is dropped where its lot is below ``round(p * 65536)``.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ELEM = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-6
SEED, CALLS = 0x1234567_89ABCDEF, 5
LOTS = 65536


def _case(name, **c):
    return {**c, "name": name} if name else c


def _norm(name, dtype, rows, width, weight="same"):
    """``weight``: the type of the norm's weight, that of the rows or fp32."""
    return _case(name, kind="norm", dtype=dtype, rows=rows, width=width, weight=weight)


def _norm_train(name, dtype, rows, width, p, weight="same"):
    return _case(name, kind="norm_train", dtype=dtype, rows=rows, width=width, p=p, weight=weight)


def _norm8_linear(name, dtype, rows, width, c_out):
    return _case(name, kind="norm8_linear", dtype=dtype, rows=rows, width=width, c_out=c_out, weight="same")


def _linear8(name, dtype, rows, groups, c_in, c_out, spread=0.5, rest=0, split=1):
    """``spread``: how unevenly the rows fall to the groups, ``rest``: rows behind the last group."""
    return _case(name, kind="linear8", dtype=dtype, rows=rows, groups=groups, c_in=c_in, c_out=c_out, spread=spread, rest=rest, split=split)


def _dropout(name, dtype, rows, width, p, residual, train):
    return _case(name, kind="dropout", dtype=dtype, rows=rows, width=width, p=p, residual=residual, train=train)


def _experts(name, dtype, tokens, experts, top_k, width, hidden, gated):
    return _case(name, kind="experts", dtype=dtype, tokens=tokens, experts=experts, top_k=top_k, width=width, hidden=hidden, gated=gated)


def listed():
    return [
        # a long prompt, or a training batch's forward
        _norm("norm_prompt", "bf16", 16384, 4096),
        # a ragged batch in fp16, a width that no tile divides
        _norm("norm_ragged", "fp16", 5003, 1001, weight="fp32"),
        # a training step of the sum and norm between two layers, dropout on the branch
        _norm_train("norm_train", "bf16", 8192, 2048, 0.1, weight="fp32"),
        # serving, one token through the norm and the layer behind it: all latency and weights
        _norm8_linear("norm8_linear_one_token", "bf16", 1, 2048, 4096),
        # the same for a prompt
        _norm8_linear("norm8_linear_prompt", "bf16", 4096, 2048, 4096),
        # a ragged batch of a layer of experts in 8 bits, widths that no tile divides, rows behind the last group
        _linear8("linear8_ragged", "fp16", 5003, 12, 1000, 1496, spread=0.8, rest=57),
        # a long prompt through one matrix
        _linear8("linear8_large", "bf16", 16384, 1, 2048, 4096, spread=0.0),
        # a small head's features
        _dropout("dropout_small", "fp32", 100, 260, 0.5, False, False),
        # a training batch, forward and backward, with the residual's addition
        _dropout("dropout_train", "bf16", 32768, 2048, 0.1, True, True),
        # serving, one token
        _experts("experts_one_token", "bf16", 1, 8, 2, 512, 1024, True),
        # serving, a batch of single tokens over many experts: every weight is read for a token or two
        _experts("experts_tokens", "bf16", 16, 64, 4, 2048, 1024, True),
        # more tokens, experts without a gate
        _experts("experts_batch", "fp16", 64, 32, 2, 1024, 2048, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, odd=0.25):
    w = _log(rng, lo, hi)
    return w if rng.random() < odd else max(8, w // 8 * 8)


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm8_linear", "linear8", "dropout", "experts", "experts"])
    dtype = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
    if kind in ("norm", "norm_train", "dropout"):
        width = _width(rng, 64, 8192)
        rows = _log(rng, 1, min(32768, (1 << (25 if kind == "norm_train" else 26)) // width))
        if kind == "norm":
            return _norm(None, dtype, rows, width, rng.choice(["same", "fp32"]))
        p = rng.choice([0.05, 0.1, 0.2, 0.5])
        if kind == "norm_train":
            return _norm_train(None, dtype, rows, width, p, rng.choice(["same", "fp32"]))
        return _dropout(None, dtype, rows, width, p, rng.random() < 0.5, rng.random() < 0.5)
    if kind == "norm8_linear":
        return _norm8_linear(None, dtype, _log(rng, 1, 4096), _width(rng, 64, 4096), _width(rng, 64, 4096))
    if kind == "linear8":
        a, b = _width(rng, 64, 4096), _width(rng, 64, 4096)
        groups = _log(rng, 1, 64)
        while groups * a * b > 1 << 27:
            groups //= 2
        rows = _log(rng, 1, max(2, min(16384, int(2.5e11 / (2.0 * a * b)))))
        return _linear8(None, dtype, rows, groups, a, b, round(rng.uniform(0, 1), 2), rng.choice([0, 0, rng.randrange(1, 200)]), rng.randrange(1 << 30))
    experts = _log(rng, 4, 64)
    a, b = _width(rng, 128, 2048, 0.0), _width(rng, 128, 2048, 0.0)
    while experts * a * b > 1 << 27:
        experts //= 2
    return _experts(None, rng.choice(["bf16", "fp16"]), _log(rng, 1, 64), experts, rng.randrange(1, min(8, experts) + 1), a, b, rng.random() < 0.7)


def sizes(case):
    """Rows of every group: ``rows`` shared out in proportion to weights that are log-normal, the remainder at random."""
    rng = random.Random(case["split"])
    share = [math.exp(rng.gauss(0, 1) * case["spread"]) for _ in range(case["groups"])]
    total = sum(share)
    n = [int(case["rows"] * s / total) for s in share]
    for _ in range(case["rows"] - sum(n)):
        n[rng.choices(range(case["groups"]), weights=share)[0]] += 1
    return n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPE[case["dtype"]], case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def codes(*shape):
        """Whole numbers in 8 bits, rows a multiple of 16 bytes apart, as ``nn.quantize_rows`` lays them out."""
        width = shape[-1]
        room = torch.empty((*shape[:-1], (width + 15) // 16 * 16), dtype=torch.int8, device="cuda")
        room.copy_((normal(*room.shape) * 32).round().clamp(-127, 127))
        return room[..., :width]

    def scales(*shape):
        return torch.exp(normal(*shape) * 0.5) * 0.01

    s = {"kind": kind, "dtype": dtype}
    if kind in ("norm", "norm_train", "norm8_linear"):
        rows, width = case["rows"], case["width"]
        s["x"] = normal(rows, width).to(dtype)
        s["residual"] = (normal(rows, width) * torch.exp(normal(rows, 1))).to(dtype)  # rows differ in size
        s["weight"] = (1 + 0.2 * normal(width)).to(dtype if case["weight"] == "same" else torch.float32)
    if kind == "norm_train":
        s["p"], s["rng"] = case["p"], torch.tensor([SEED, CALLS, 0], dtype=torch.int64, device="cuda")
        for name in ("x", "residual", "weight"):
            s[name].requires_grad_()
        s["out_grad"], s["sum_grad"] = normal(rows, width).to(dtype), normal(rows, width).to(dtype)
    if kind == "norm8_linear":
        s["kernel"], s["kernel_scale"] = codes(1, case["c_out"], width), scales(1, case["c_out"])
    if kind == "linear8":
        n, kpos = sizes(case), [0]
        for k in n:
            kpos.append(kpos[-1] + k)
        rows = case["rows"] + case["rest"]
        s["sizes"], s["kpos"] = n, torch.tensor(kpos, dtype=torch.int32, device="cuda")
        s["codes"], s["scale"] = codes(rows, case["c_in"]), scales(rows)
        s["scale"][case["rows"]:] = math.nan  # whatever a buffer with room to spare holds behind its rows
        s["kernel"], s["kernel_scale"] = codes(case["groups"], case["c_out"], case["c_in"]), scales(case["groups"], case["c_out"])
        s["out"] = torch.full((rows, case["c_out"]), 0.5, dtype=dtype, device="cuda")
    if kind == "dropout":
        rows, width = case["rows"], case["width"]
        s["p"], s["rng"] = case["p"], torch.tensor([SEED, CALLS, 0], dtype=torch.int64, device="cuda")
        s["x"] = normal(rows, width).to(dtype).requires_grad_(case["train"])
        s["residual"] = normal(rows, width).to(dtype) if case["residual"] else None
        s["out_grad"] = normal(rows, width).to(dtype) if case["train"] else None
    if kind == "experts":
        t, e, a, b = case["tokens"], case["experts"], case["width"], case["hidden"]
        s["gated"], s["top_k"] = case["gated"], case["top_k"]
        s["x"], s["router"] = normal(t, a).to(dtype), (normal(e, a) * a ** -0.5).to(dtype)
        s["w_in"] = (normal(e, a, (2 if case["gated"] else 1) * b) * a ** -0.5).to(dtype)
        s["w_out"] = (normal(e, b, a) * b ** -0.5).to(dtype)
        s["out"] = torch.empty((t, a), dtype=dtype, device="cuda")
        s["experts"] = torch.empty((t, case["top_k"]), dtype=torch.int32, device="cuda")
        s["gates"] = torch.empty((t, case["top_k"]), dtype=torch.float32, device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _times(a, b):
    """The two halves of the 64-bit product of numbers of 32 bits (held in 64): its high half is what stands above bit 31, wrapped or not."""
    wide = a * b
    return (wide >> 32) & 0xFFFFFFFF, wide & 0xFFFFFFFF


def _keep(rng, rows, width, p):
    """Which values of ``rows`` by ``width`` the next call keeps, and what they are multiplied by."""
    seed, call = rng[0], rng[1]
    key0, key1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    blocks = (width + 7) // 8
    c0 = torch.arange(blocks, device="cuda").expand(rows, blocks)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, blocks)
    c2, c3 = (call & 0xFFFFFFFF).expand(rows, blocks), ((call >> 32) & 0xFFFFFFFF).expand(rows, blocks)
    for _ in range(10):
        hi0, lo0 = _times(c0, 0xD2511F53)
        hi1, lo1 = _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = hi1 ^ c1 ^ key0, lo1, hi0 ^ c3 ^ key1, lo0
        key0, key1 = (key0 + 0x9E3779B9) & 0xFFFFFFFF, (key1 + 0xBB67AE85) & 0xFFFFFFFF
    lots = torch.stack([c & 0xFFFF if half == 0 else c >> 16 for c in (c0, c1, c2, c3) for half in (0, 1)], -1).view(rows, blocks * 8)[:, :width]
    threshold = round(p * LOTS)
    return lots >= threshold, LOTS / (LOTS - threshold)


def _plain_sum_and_norm(h, weight):
    return h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * weight.detach().float()


def _plain_norm_train(s):
    x, residual, w = s["x"].detach().float(), s["residual"].detach().float(), s["weight"].detach().float()
    keep, factor = _keep(s["rng"], *x.shape, s["p"])
    s["rng"][1] += 1
    h = residual + torch.where(keep, x * factor, 0.0)
    r = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    normed, dy = h * r, s["out_grad"].float()
    g = dy * w
    dh = r * (g - normed * (g * normed).mean(1, keepdim=True)) + s["sum_grad"].float()
    return {"out": (normed * w).to(s["dtype"]), "sum": h.to(s["dtype"]), "x_grad": torch.where(keep, dh * factor, 0.0).to(s["dtype"]),
            "residual_grad": dh.to(s["dtype"]), "weight_grad": (dy * normed).sum(0).to(s["weight"].dtype)}


def _plain_norm8_linear(s):
    h = s["x"].float() + s["residual"].float()
    y = _plain_sum_and_norm(h, s["weight"])
    scale = y.abs().amax(1) / 127.0
    code = (y / scale.clamp(min=1e-30)[:, None]).round().clamp(-127, 127)
    out = code @ s["kernel"][0].float().T * scale[:, None] * s["kernel_scale"][0]
    return {"out": out.to(s["dtype"]), "sum": h.to(s["dtype"])}


def _plain_linear8(s):
    at = 0
    for g, n in enumerate(s["sizes"]):
        rows = slice(at, at + n)
        sums = s["codes"][rows].float() @ s["kernel"][g].float().T
        s["out"][rows] = (sums * s["scale"][rows, None] * s["kernel_scale"][g]).to(s["dtype"])
        at += n
    return s["out"]


def _plain_dropout(s):
    x = s["x"].detach().float()
    keep, factor = _keep(s["rng"], *x.shape, s["p"])
    s["rng"][1] += 1
    out = torch.where(keep, x * factor, 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    result = {"out": out.to(s["dtype"])}
    if s["out_grad"] is not None:
        result["x_grad"] = torch.where(keep, s["out_grad"].float() * factor, 0.0).to(s["dtype"])
    return result


def _plain_experts(s):
    x = s["x"].float()
    logits = s["x"].double() @ s["router"].double().T  # a choice hangs on the difference of two of them
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)
    chosen, value = order[:, :s["top_k"]], value[:, :s["top_k"]]
    gate = torch.exp(value - value[:, :1])
    gate = (gate / gate.sum(1, keepdim=True)).float()
    share = torch.zeros(logits.shape, device="cuda").scatter_(1, chosen, gate)  # [tokens, experts]
    u = torch.bmm(x.expand(share.size(1), -1, -1), s["w_in"].float())  # every expert on every token
    if s["gated"]:
        a, b = u.chunk(2, 2)
        h = a / (1.0 + torch.exp(-a)) * b
    else:
        h = u.clamp(min=0.0)
    out = torch.bmm(h * share.T[:, :, None], s["w_out"].float()).sum(0)
    return {"out": out.to(s["dtype"]), "experts": chosen.int(), "gates": gate}


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if own:
        from fgms_b200 import backend, nn
        if kind == "norm":
            out, total = nn.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
            return {"out": out, "sum": total}
        if kind == "norm_train":
            out, total = nn.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], dropout=s["p"], rng=s["rng"])
            grads = torch.autograd.grad((out, total), (s["x"], s["residual"], s["weight"]), (s["out_grad"], s["sum_grad"]))
            return {"out": out.detach(), "sum": total.detach(), "x_grad": grads[0], "residual_grad": grads[1], "weight_grad": grads[2]}
        if kind == "norm8_linear":
            codes, scale, total = nn.rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
            return {"out": nn.int8_linear(codes, scale, s["kernel"], s["kernel_scale"], dtype=s["dtype"]), "sum": total}
        if kind == "linear8":
            backend.fgms_grouped_i8_fwd_cuda(s["codes"], s["scale"], s["kernel"], s["kernel_scale"], s["out"], s["kpos"])
            return s["out"]
        if kind == "dropout":
            out = nn.dropout(s["x"], s["p"], s["rng"], residual=s["residual"])
            if s["out_grad"] is None:
                return {"out": out}
            return {"out": out.detach(), "x_grad": torch.autograd.grad(out, s["x"], s["out_grad"])[0]}
        backend.fgms_expert_layer_cuda(s["x"], s["router"], s["w_in"], s["w_out"], s["out"], s["experts"], s["gates"],
                                       activation="silu" if s["gated"] else "relu")
        return {"out": s["out"], "experts": s["experts"], "gates": s["gates"]}
    if kind == "norm":
        h = s["x"].float() + s["residual"].float()
        return {"out": _plain_sum_and_norm(h, s["weight"]).to(s["dtype"]), "sum": h.to(s["dtype"])}
    return {"norm_train": _plain_norm_train, "norm8_linear": _plain_norm8_linear, "linear8": _plain_linear8, "dropout": _plain_dropout,
            "experts": _plain_experts}[kind](s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def _used(case):
    """Experts that some token goes to, on average, where every choice is as likely as any other."""
    e, k = case["experts"], case["top_k"]
    return e * (1.0 - (1.0 - k / e) ** case["tokens"])


def work(case):
    kind, e = case["kind"], ELEM[case["dtype"]]
    if kind in ("norm", "norm_train", "dropout"):
        n = float(case["rows"] * case["width"])
        if kind == "norm":
            return {"bytes": 4 * n * e + case["width"] * e, "flops": 5 * n}
        if kind == "norm_train":  # forward as above; backward: both gradients and the sum in, two gradients out
            return {"bytes": (4 + 5) * n * e + case["width"] * 8, "flops": 20 * n}
        return {"bytes": n * e * (2 + case["residual"] + 2 * case["train"]), "flops": 3 * n}
    if kind == "norm8_linear":
        r, a, b = float(case["rows"]), case["width"], case["c_out"]
        return {"bytes": r * (3 * a + b) * e + float(a * b) + 4 * b, "flops": 2 * r * a * b}
    if kind == "linear8":
        n, a, b = sizes(case), case["c_in"], case["c_out"]
        r, used = float(sum(n)), float(sum(k > 0 for k in n))
        return {"bytes": r * (a + 4 + b * e) + used * (a + 4) * b, "flops": 2 * r * a * b}
    t, a, b = case["tokens"], case["width"], case["hidden"]
    matrices = float(a * b) * (3 if case["gated"] else 2)
    return {"bytes": e * (_used(case) * matrices + case["experts"] * a + 2 * t * a), "flops": 2 * t * (case["top_k"] * matrices + case["experts"] * a)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _mask(case):
    """Philox once more, in unsigned numbers of 64 bits on the host."""
    rows, width, blocks = case["rows"], case["width"], (case["width"] + 7) // 8
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    ctr = [np.broadcast_to(np.arange(blocks, dtype=np.uint64), (rows, blocks)), np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, blocks)),
           np.full((rows, blocks), CALLS & 0xFFFFFFFF, np.uint64), np.full((rows, blocks), CALLS >> 32, np.uint64)]
    key = [SEED & 0xFFFFFFFF, SEED >> 32]
    for _ in range(10):
        first, second = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(second >> half) ^ ctr[1] ^ np.uint64(key[0]), second & low, (first >> half) ^ ctr[3] ^ np.uint64(key[1]), first & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(ctr, -1).astype(np.uint32)  # little-endian: the lower half of a word is the earlier column's lot
    lots = words.view(np.uint16).reshape(rows, blocks * 8)[:, :width]
    threshold = round(case["p"] * LOTS)
    return torch.from_numpy(lots >= threshold).cuda().double() * (LOTS / (LOTS - threshold))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    get = lambda name: s[name].detach().double()
    if kind == "dropout":
        mask = _mask(case)
        out = get("x") * mask + (get("residual") if case["residual"] else 0.0)
        return {"out": out, "x_grad": get("out_grad") * mask} if case["train"] else {"out": out}
    if kind in ("norm", "norm_train", "norm8_linear"):
        mask = _mask(case) if kind == "norm_train" else 1.0
        h, w = get("residual") + get("x") * mask, get("weight")
        root = (h.square().sum(1, keepdim=True) / case["width"] + EPS).sqrt()
        y = h / root * w
        if kind == "norm":
            return {"out": y, "sum": h}
        if kind == "norm8_linear":
            scale = y.abs().amax(1, keepdim=True) / 127
            return {"out": torch.round(y / scale) * scale @ (get("kernel")[0] * get("kernel_scale")[0][:, None]).T, "sum": h}
        dy = get("out_grad")
        dh = dy * w / root - h * (dy * w * h).sum(1, keepdim=True) / (case["width"] * root ** 3) + get("sum_grad")
        return {"out": y, "sum": h, "x_grad": dh * mask, "residual_grad": dh, "weight_grad": (dy * h / root).sum(0)}
    if kind == "linear8":
        out, at = torch.full(s["out"].shape, 0.5, dtype=torch.float64, device="cuda"), 0
        for g, n in enumerate(s["sizes"]):
            a = get("codes")[at:at + n] * get("scale")[at:at + n, None]
            out[at:at + n] = a @ (get("kernel")[g] * get("kernel_scale")[g][:, None]).T
            at += n
        return out
    x, top_k = get("x"), case["top_k"]
    logits = (x[:, None, :] * get("router")[None]).sum(2)
    out, chosen, gates = torch.zeros_like(x), [], []
    for t, row in enumerate(logits.tolist()):
        picked = sorted(range(len(row)), key=lambda e: (-row[e], e))[:top_k]
        total = sum(math.exp(row[e] - row[picked[0]]) for e in picked)
        chosen.append(picked)
        gates.append([math.exp(row[e] - row[picked[0]]) / total for e in picked])
        for e, gate in zip(picked, gates[-1]):
            u = x[t] @ s["w_in"][e].double()
            h = u[:case["hidden"]] * torch.sigmoid(u[:case["hidden"]]) * u[case["hidden"]:] if case["gated"] else torch.relu(u)
            out[t] += gate * (h @ s["w_out"][e].double())
    return {"out": out, "experts": torch.tensor(chosen, dtype=torch.int32, device="cuda"), "gates": torch.tensor(gates, dtype=torch.float64, device="cuda")}
