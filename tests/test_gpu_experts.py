"""A layer of experts for a few tokens against its definition in 64 bits, and the layer of any number of tokens around it.

What is allowed, to the first order: a sum of n products in fp32 is off by (n + 1) 2^-23 of the sum of the magnitudes; an activation has a slope of 1.1 at
most and is itself off by 2^-20 of its value (its exponential by 2^-21); h is the sum of two values of its type, off by half a step of half a step; a gate is off by 2^-18 (logits in 64
bits, their difference, at most 32 here, rounded to fp32, so 2^-19 of its exponential); the output is rounded once more."""
import pytest
import torch

from tests.layers_ref import near, tiny

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Layer:
    def __init__(self, dtype, tokens, experts, top_k, width, hidden, out_width=None, gated=True, seed=0, router_type=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(s, generator=gen, device="cuda")
        t = TYPES[dtype]
        out_width = out_width or width
        self.gated, self.top_k, self.type = gated, top_k, t
        self.x, self.router = normal(tokens, width).to(t), (normal(experts, width) * width ** -0.5).to(router_type or t)
        self.w_in = (normal(experts, width, (2 if gated else 1) * hidden) * width ** -0.5).to(t)
        self.w_out = (normal(experts, hidden, out_width) * hidden ** -0.5).to(t)

    def run(self, activation="silu", x=None, out=None):
        from fgms_b200 import backend
        x = self.x if x is None else x
        out = torch.full((x.size(0), self.w_out.size(2)), float("nan"), dtype=self.type, device="cuda") if out is None else out
        experts = torch.full((x.size(0), self.top_k), -1, dtype=torch.int32, device="cuda")
        gates = torch.full((x.size(0), self.top_k), float("nan"), device="cuda")
        backend.fgms_expert_layer_cuda(x, self.router, self.w_in, self.w_out, out, experts, gates, activation=activation)
        return out, experts, gates

    def exact(self, activation="silu"):
        """(out, allowed, experts, gates)"""
        x, unit = self.x.double(), torch.finfo(self.type).eps / 2
        logits = x @ self.router.double().T
        value, chosen = (v[:, :self.top_k] for v in torch.sort(logits, dim=1, descending=True, stable=True))
        gates = torch.softmax(value, 1)
        out = torch.zeros((x.size(0), self.w_out.size(2)), dtype=torch.float64, device="cuda")
        off = torch.zeros_like(out)
        hidden = self.w_out.size(1)
        for e in chosen.unique().tolist():
            token, j = (chosen == e).nonzero(as_tuple=True)
            w, v, rows = self.w_in[e].double(), self.w_out[e].double(), x[token]
            u, du = rows @ w, (rows.abs() @ w.abs()) * ((w.size(0) + 1) * 2.0 ** -23)
            a, da = u[:, :hidden], du[:, :hidden]
            act = a * torch.sigmoid(a) if activation == "silu" else a.clamp(min=0)
            da = 1.1 * da + act.abs() * 2.0 ** -20
            h, dh = act, da
            if self.gated:
                b, db = u[:, hidden:], du[:, hidden:]
                h, dh = act * b, da * b.abs() + act.abs() * db + da * db
            dh = dh * (1 + 2 * unit) + h.abs() * unit * unit + tiny(self.type)  # h: its rounding and the rounded remainder
            y = h @ v
            dy = dh @ v.abs() + (h.abs() + dh) @ v.abs() * ((hidden + 1) * 2.0 ** -23)
            g = gates[token, j][:, None]
            out.index_add_(0, token, g * y)
            off.index_add_(0, token, g * (dy + (y.abs() + dy) * 2.0 ** -18))
        return out, off * (1 + unit) + out.abs() * (unit + self.top_k * 2.0 ** -23) + tiny(self.type), chosen.int(), gates

    def check(self, got, activation="silu"):
        from fgms_b200 import backend
        out, allowed, chosen, gates = self.exact(activation)
        assert torch.equal(got[1], chosen)
        near(got[2], gates, gates * 2.0 ** -18 + 1e-30)
        near(got[0], out, allowed)
        assert backend.device_status() == 0


# tokens, experts, top_k, width, hidden, out_width, gated
CASES = [
    (1, 1, 1, 8, 8, 8, True), (1, 4, 2, 64, 64, 64, True), (1, 8, 2, 512, 1024, 512, True), (1, 8, 8, 128, 72, 136, False), (2, 5, 3, 40, 200, 24, True),
    (7, 512, 16, 256, 64, 256, True), (8, 16, 1, 72, 136, 72, False), (9, 3, 3, 200, 264, 520, True), (17, 64, 4, 512, 256, 512, True), (18, 2, 1, 1032, 64, 8, True),
    (19, 33, 5, 96, 96, 96, False), (33, 300, 7, 128, 128, 128, True), (64, 1, 1, 256, 512, 256, True), (64, 4, 4, 520, 328, 264, False), (64, 32, 2, 1024, 2048, 1024, False),
    (64, 64, 16, 64, 64, 64, True), (40, 20, 6, 8, 4096, 8, True), (3, 6, 2, 4096, 8, 4096, True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(case, dtype):
    tokens, experts, top_k, width, hidden, out_width, gated = CASES[case]
    layer = Layer(dtype, tokens, experts, top_k, width, hidden, out_width, gated, seed=case, router_type=torch.float32 if case % 3 == 0 else None)
    for activation in ("silu", "relu"):
        layer.check(layer.run(activation), activation)
    first = layer.run()
    assert all(torch.equal(a, b) for a, b in zip(first, layer.run()))


@pytest.mark.parametrize("tokens", range(1, 65))
def test_every_number_of_tokens_that_an_expert_may_have(tokens):
    """The rings in shared memory are cut by it (``test_expert_rings_cpu.py`` has their sizes): all tokens to the first of two experts."""
    layer = Layer("bf16", tokens, 2, 1, 264, 200, seed=tokens)
    layer.router[1] = layer.router[0]
    layer.check(layer.run())


def test_equal_logits_go_to_the_lower_index():
    layer = Layer("bf16", 30, 40, 6, 64, 64, seed=2)
    layer.router[7:33] = layer.router[5]
    layer.check(layer.run())
    layer.router.zero_()
    got = layer.run()
    assert torch.equal(got[1], torch.arange(6, dtype=torch.int32, device="cuda").expand(30, 6)) and (got[2] == torch.tensor(1 / 6)).all()
    layer.check(got)


def test_logits_that_differ_by_less_than_fp32_tells():
    """Two experts whose logits differ in the 40th bit, the larger one last."""
    layer = Layer("fp16", 1, 8, 1, 4096, 64, seed=3, router_type=torch.float32)
    layer.x.fill_(1.0)
    layer.router.zero_()
    layer.router[:, 0] = 2.0 ** 20
    layer.router[6, 4095] = 2.0 ** -20
    got = layer.run()
    assert got[1].item() == 6
    layer.check(got)


def test_tokens_that_are_not_finite_stay_by_themselves():
    layer = Layer("bf16", 20, 8, 2, 128, 128, seed=4)
    want = layer.run()
    layer.x[3, 5], layer.x[11] = float("nan"), float("inf")
    got = layer.run()
    rest = [t for t in range(20) if t not in (3, 11)]
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, want))
    assert torch.isnan(got[0][[3, 11]]).all() and torch.isnan(got[2][3]).all()
    assert ((got[1] >= 0) & (got[1] < 8)).all()


def test_in_place_strides_and_no_tokens():
    from fgms_b200 import backend
    layer = Layer("bf16", 12, 8, 2, 64, 96, seed=5)
    want = layer.run()
    wide = torch.zeros((12, 200), dtype=torch.bfloat16, device="cuda")
    x, out = wide[:, :64], wide[:, 67:131]  # out off every boundary
    x.copy_(layer.x)
    got = layer.run(x=x, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (wide[:, 64:67] == 0).all() and (wide[:, 131:] == 0).all() and torch.equal(x, layer.x)
    x = layer.x.clone()
    assert torch.equal(layer.run(x=x, out=x)[0], want[0])
    empty = torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda")
    assert layer.run(x=empty)[0].shape == (0, 64) and backend.device_status() == 0


def test_on_a_stream_and_in_two_graphs():
    layers = [Layer("bf16", 30, 16, 3, 256, 256, seed=6), Layer("bf16", 5, 16, 2, 256, 192, seed=7)]
    want = [l.run() for l in layers]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [l.run() for l in layers]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    graphs, got = [], []
    for l in layers:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(l.run())
    for _ in range(3):
        for g in graphs:
            g.replay()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
        for l in layers:
            l.x.mul_(-1)
        want = [l.run() for l in layers]


def test_one_call_behind_the_other_on_two_streams():
    layers = [Layer("bf16", 64, 16, 3, 256, 512, seed=s) for s in (8, 9)]
    want = [l.run() for l in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(6):
        for i, (l, st) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(st):
                got[i] = l.run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_with_sms_kept_free():
    from fgms_b200 import _lib
    layer = Layer("fp16", 25, 16, 3, 256, 320, seed=10)
    for n in (20, 64):
        _lib.lib.fgms_b200_set_reserved_sms(n)
        try:
            got = layer.run()
        finally:
            _lib.lib.fgms_b200_set_reserved_sms(0)
        layer.check(got)


def reference(x, router, w_in, w_out, top_k, activation):
    """The layer and its autograd in 64 bits, every expert on every row."""
    logits = x @ router.T
    value, chosen = (v[:, :top_k] for v in torch.sort(logits, dim=1, descending=True, stable=True))
    share = torch.zeros_like(logits).scatter(1, chosen, torch.softmax(value, 1))
    u = torch.einsum("tc,ech->eth", x, w_in)
    act = (lambda v: v * torch.sigmoid(v)) if activation == "silu" else torch.relu
    hidden = w_out.size(1)
    h = act(u[..., :hidden]) * u[..., hidden:] if u.size(2) == 2 * hidden else act(u)
    return torch.einsum("eth,eho,te->to", h, w_out, share)


@pytest.mark.parametrize("gated,activation", [(True, "silu"), (False, "relu")])
def test_a_layer_of_any_number_of_rows_and_its_gradients(gated, activation):
    """fp32 through the grouped products; every value within 2^-12 of the largest: sums of at most 200 products, four in a row, each off by 2^-15.3 of the sum of
    the magnitudes, which for values like these is at most a few times the largest value."""
    from fgms_b200 import nn
    gen = torch.Generator(device="cuda").manual_seed(11)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda")
    x, router = normal(2, 75, 48), normal(6, 48) * 48 ** -0.5
    w_in, w_out = normal(6, 48, 2 * 56 if gated else 56) * 48 ** -0.5, normal(6, 56, 40) * 56 ** -0.5
    leaves = [t.requires_grad_() for t in (x, router, w_in, w_out)]
    out = nn.expert_layer(*leaves, 2, activation)
    g = normal(2, 75, 40)
    grads = torch.autograd.grad(out, leaves, g)
    double = [t.detach().double().requires_grad_() for t in leaves]
    want = reference(double[0].view(150, 48), *double[1:], 2, activation)
    exact = torch.autograd.grad(want, double, g.double().view(150, 40))
    for got, ref in zip((out.detach().view(150, 40), *grads), (want.detach(), *exact)):
        assert (got.double() - ref).abs().max() <= 2.0 ** -12 * ref.abs().max()


def test_both_ways_give_the_same_layer():
    """Rows that need no gradient go through the kernel for a few tokens, others through the grouped products."""
    from fgms_b200 import backend, nn
    layer = Layer("bf16", 40, 8, 2, 128, 192, seed=12)
    module = nn.ExpertLayer(128, 192, 8, 2)
    with torch.no_grad():
        for name in ("router", "w_in", "w_out"):
            getattr(module, name).copy_(getattr(layer, name))
    routed = module(layer.x)
    assert routed.requires_grad
    before = backend.launch_count()
    with torch.no_grad():
        few = module(layer.x.view(4, 10, 128))
    assert backend.launch_count() - before == 2 and few.shape == (4, 10, 128)
    out, allowed, _, _ = layer.exact()
    near(few.view(40, 128), out, allowed)
    # There u, h and the experts' outputs are each rounded to 8 bits as well.  h is off by 3.2 half steps of its size then (u in both factors, the activation's slope, itself),
    # the output by that of the sum of the magnitudes of what it is added up from, and by one more half step of each expert's part.
    x = layer.x.double()
    share = torch.zeros((40, 8), dtype=torch.float64, device="cuda").scatter_(1, layer.exact()[2].long(), layer.exact()[3])
    u = torch.einsum("tc,ech->teh", x, layer.w_in.double())
    size = torch.einsum("teh,eho,te->to", (1.1 * u[..., :192].abs() * u[..., 192:].abs()), layer.w_out.double().abs(), share)
    near(routed.detach(), out, allowed + 4.5 * 2.0 ** -8 * size)
    with torch.no_grad():
        assert torch.equal(module(layer.x.repeat(2, 1))[:40], module(layer.x.repeat(2, 1))[40:])
        assert module(layer.x[:0]).shape == (0, 128) and module(layer.x[0]).shape == (128,)
        assert torch.equal(module(layer.x[0]), few.view(40, 128)[0])
        fp16 = nn.expert_layer(layer.x, module.router.half(), module.w_in, module.w_out, 2)  # a router of another 16-bit type: not through the kernel
        assert (fp16.float() - few.view(40, 128).float()).abs().max() < 1.0


def test_a_block_in_training_and_in_serving():
    """Norm with the residual's addition, experts, dropout: a training step has finite gradients everywhere, and without dropout and gradients the block is the
    sum of its parts."""
    from fgms_b200 import nn
    gen = torch.Generator(device="cuda").manual_seed(13)
    x, res = (torch.randn((60, 64), generator=gen, device="cuda").bfloat16() for _ in range(2))
    norm, experts, drop = nn.RMSNorm(64, dropout=0.1), nn.ExpertLayer(64, 128, 8, 2), nn.Dropout(0.2, seed=3)

    def block(x, res):
        y, h = norm(x, res)
        return drop(experts(y), h)

    x.requires_grad_(), res.requires_grad_()
    out = block(x, res)
    params = [x, res, norm.weight, *experts.parameters()]
    grads = torch.autograd.grad(out.float().square().sum(), params)
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)
    for m in (norm, experts, drop):
        m.eval()
    with torch.no_grad():
        y, h = nn.rms_norm(x, norm.weight, residual=res)
        assert torch.equal(block(x, res), h + nn.expert_layer(y, experts.router, experts.w_in, experts.w_out, 2))


def test_refusals():
    from fgms_b200 import backend, nn
    layer = Layer("bf16", 6, 8, 2, 64, 96)
    a = dict(x=layer.x, router=layer.router, w_in=layer.w_in, w_out=layer.w_out, out=torch.zeros_like(layer.x), experts=torch.zeros((6, 2), dtype=torch.int32, device="cuda"),
             gates=torch.zeros((6, 2), device="cuda"))
    big = torch.zeros((65, 64), dtype=torch.bfloat16, device="cuda")
    for change, text in [
        (dict(x=layer.x.float()), "dtype"), (dict(x=layer.x[:, :32]), "channels"), (dict(x=layer.x.cpu()), "CUDA"), (dict(w_in=layer.w_in.half()), "dtype"),
        (dict(w_in=layer.w_in[:, :, :100].contiguous()), "twice"), (dict(w_out=layer.w_out[:4]), "differ in experts"), (dict(router=layer.router[:, :60].contiguous()), "channels"),
        (dict(router=layer.router.half()), "router's type"), (dict(out=torch.zeros((6, 60), device="cuda")), "out must be"), (dict(experts=a["experts"].long()), "int32"),
        (dict(gates=a["gates"][:, :1]), "gates"), (dict(experts=a["experts"][:5]), "experts must be"), (dict(activation="tanh"), "activation"),
        (dict(experts=torch.zeros((6, 9), dtype=torch.int32, device="cuda"), gates=torch.zeros((6, 9), device="cuda")), "top_k 9"),
        (dict(x=big, out=big.clone(), experts=torch.zeros((65, 2), dtype=torch.int32, device="cuda"), gates=torch.zeros((65, 2), device="cuda")), "tokens 65"),
        (dict(out=layer.w_out[0, :6]), "overlaps"), (dict(w_in=layer.w_in.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
        (dict(x=torch.zeros(6 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 64)), "16-byte"),
    ]:
        with pytest.raises(ValueError, match=text):
            backend.fgms_expert_layer_cuda(**{**a, **change})
    for args, text in [((layer.x, layer.router[:7], layer.w_in, layer.w_out, 2), "same experts"), ((layer.x, layer.router, layer.w_in, layer.w_out, 9), "top_k"),
                       ((layer.x, layer.router, layer.w_in[:, :, :50], layer.w_out, 2), "twice"), ((layer.x, layer.router, layer.w_in, layer.w_out, 2, "gelu"), "activation")]:
        with pytest.raises(ValueError, match=text):
            nn.expert_layer(*args)
