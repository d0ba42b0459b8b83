"""AdamW over many tensors against its formulas in 64 bits.

Allowed differences.  fp32 arithmetic, every operation off by half a step (2^-24 of its result) at most, constants rounded once more:
a moment is two products and a sum, four roundings of no more than the sum of its terms' absolute values: 2^-22 of that.  The update is
rate * m / (sqrt(v) * root + eps), seven roundings of its own (rate, root, sqrt, two products, sum, quotient), of which v's own error enters
halved: 2^-20 of rate * (terms of m) / denominator.  The new value is a product and a difference: 2^-22 of |w| more.  What is held in 16
bits: half a step of that type more.  Codes of 8 bits are the neighbours, below and above, of value / scale, both of which are off by a moment's
error: relative to the value's own terms, which may cancel, not to what is left of them.  On top of that come three roundings (scale,
its inverse, the product): 2^-21 of the scale, 2^-20 of the quotient."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LR, B1, B2, EPS, DECAY = 2e-3, 0.9, 0.999, 1e-8, 0.02
COUNTS = [1, 7, 0, 127, 128, 129, 2047, 2048, 2049, 100003]


def blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % 128)).view(-1, 128)


def held(code, scale):
    return (blocks(code.float()).double() * scale.double()[:, None]).view(-1)[:code.numel()].view(code.shape)


class State:
    def __init__(self, counts=COUNTS, param="fp32", grad=None, master=False, bits=32, seed=0, shift=0, steps=4, size=1e-2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda n: torch.randn(n, generator=gen, device="cuda")

        def place(x):
            """The values in a buffer that starts `shift` values off a boundary."""
            flat = torch.empty(x.numel() + shift, dtype=x.dtype, device="cuda")
            flat[shift:].copy_(x)
            return flat[shift:]
        self.bits = bits
        self.p = [place((normal(n) * 0.1).to(TYPES[param])) for n in counts]
        self.g = [place((normal(n) * size).to(TYPES[grad or param])) for n in counts]
        self.master = [place(p.float() + normal(p.numel()) * 1e-7) for p in self.p] if master else None
        m, v = [normal(n) * size for n in counts], [(normal(n) * size).square() for n in counts]
        if bits == 32:
            self.m, self.v, self.ms, self.vs = [place(x) for x in m], [place(x) for x in v], None, None
        else:
            scaled = lambda x, s: (blocks(x) / s.clamp(min=1e-30)[:, None]).clamp(-448, 448).view(-1)[:x.numel()].to(torch.float8_e4m3fn)
            self.ms, self.vs = [blocks(x).abs().amax(1) / 448 for x in m], [blocks(x).amax(1) / 448 for x in v]
            self.m = [place(scaled(x, s).view(torch.uint8)).view(torch.float8_e4m3fn) for x, s in zip(m, self.ms)]
            self.v = [place(scaled(x, s).view(torch.uint8)).view(torch.float8_e4m3fn) for x, s in zip(v, self.vs)]
        self.step = torch.tensor([steps, 0], dtype=torch.int32, device="cuda")

    def all(self):
        return [t for k in ("p", "g", "master", "m", "v", "ms", "vs") for t in (getattr(self, k) or [])] + [self.step]

    def run(self, lr=LR, **kw):
        from fgms_b200 import backend
        backend.fgms_adamw_cuda(self.p, self.g, self.m, self.v, self.step, lr, B1, B2, EPS, DECAY, masters=self.master, exp_avg_scales=self.ms,
                                exp_avg_sq_scales=self.vs, **kw)

    def moments(self):
        if self.bits == 32:
            return [m.double() for m in self.m], [v.double() for v in self.v]
        return [held(m, s) for m, s in zip(self.m, self.ms)], [held(v, s) for v, s in zip(self.v, self.vs)]

    def expect(self, scale=1.0, lr=LR):
        """What a step gives in 64 bits, from the state as it is: [(w, allowed, m, allowed, v, allowed)]."""
        t = int(self.step[0]) + 1
        out = []
        for i, (m, v) in enumerate(zip(*self.moments())):
            g = self.g[i].double() / scale
            w = (self.master[i] if self.master else self.p[i]).double()
            terms = B1 * m.abs() + (1 - B1) * g.abs()
            m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
            rate, denominator = lr / (1 - B1 ** t), (v / (1 - B2 ** t)).sqrt() + EPS
            new = w * (1 - lr * DECAY) - rate * m / denominator
            tiny = 2.0 ** -149
            out.append((new, w.abs() * 2.0 ** -22 + rate * terms / denominator * 2.0 ** -20 + tiny, m, terms * 2.0 ** -22 + tiny, v, v * 2.0 ** -22 + tiny))
        return out

    def check(self, expected):
        for i, (w, dw, m, dm, v, dv) in enumerate(expected):
            if self.master:
                assert ((self.master[i].double() - w).abs() <= dw).all()
                assert torch.equal(self.p[i], self.master[i].to(self.p[i].dtype))
            else:
                f = torch.finfo(self.p[i].dtype)
                half = w.abs() * (f.eps / 2) + f.smallest_normal * f.eps if f.bits == 16 else 0.0
                assert ((self.p[i].double() - w).abs() <= dw + half + dw * f.eps).all()
            if self.bits == 32:
                assert ((self.m[i].double() - m).abs() <= dm).all() and ((self.v[i].double() - v).abs() <= dv).all()
                continue
            for code, scale, x, dx, floor in ((self.m[i], self.ms[i], m, dm, False), (self.v[i], self.vs[i], v, dv, True)):
                if x.numel() == 0:
                    continue
                top = blocks(x).abs().amax(1)
                dx = blocks(dx)
                assert ((scale.double() * 448 - top).abs() <= dx.amax(1) + top * 2.0 ** -21).all()
                u = (blocks(x) / (top / 448).clamp(min=1e-300)[:, None]).abs()
                step = torch.where(u >= 2.0 ** -6, 2.0 ** (torch.floor(torch.log2(u.clamp(min=2.0 ** -6))) - 3), torch.full_like(u, 2.0 ** -9))
                got = blocks(code.float()).double()
                unit = (top / 448).clamp(min=1e-300)
                slack = dx / unit[:, None] + u * ((dx.amax(1) / (unit * 448))[:, None] + 2.0 ** -20)
                assert ((got.abs() - u).abs() <= step + slack + (2.0 ** -9 if floor else 0)).all()
                assert (got.abs() >= torch.floor(u / step) * step - step * (torch.floor(u / step) * step > u - slack) - slack).all()
                assert (torch.signbit(got) == torch.signbit(blocks(x)))[got != 0].all()
                if floor:
                    assert (got[blocks(x) > 0] > 0).all()


KINDS = [("fp32", None, False, 32), ("fp16", None, True, 32), ("bf16", None, False, 32), ("fp16", "fp32", True, 32), ("bf16", "fp32", False, 8),
         ("fp32", None, False, 8), ("fp16", None, True, 8), ("fp32", "bf16", False, 8)]


@pytest.mark.parametrize("param,grad,master,bits", KINDS)
def test_against_the_formulas(param, grad, master, bits):
    s = State(param=param, grad=grad, master=master, bits=bits, seed=1)
    for _ in range(3):
        want = s.expect()
        s.run()
        s.check(want)
    assert s.step.tolist() == [7, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_from_zeros(bits):
    s = State(param="fp32", bits=bits, seed=2, steps=0)
    for t in s.m + s.v:
        t.view(torch.uint8).zero_() if bits == 8 else t.zero_()
    for t in (s.ms or []) + (s.vs or []):
        t.zero_()
    want = s.expect()
    s.run()
    s.check(want)


@pytest.mark.parametrize("shift", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("bits", [32, 8])
def test_views_that_start_off_a_boundary(bits, shift):
    s = State(param="bf16", master=True, bits=bits, seed=3, shift=shift)
    want = s.expect()
    s.run()
    s.check(want)


@pytest.mark.parametrize("n", [48, 49, 400, 401, 850])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits, n):
    s = State(counts=[(i * 37) % 300 for i in range(n)], param="fp16", master=True, bits=bits, seed=4)
    want = s.expect()
    s.run()
    s.check(want)
    assert s.step.tolist() == [5, 0]


def test_no_tensors_still_count_the_step():
    s = State(counts=[])
    s.run()
    assert s.step.tolist() == [5, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_loss_scale_and_verdict(bits):
    s = State(param="fp16", master=True, bits=bits, seed=5, size=1.0)
    scale, fine, bad = (torch.tensor([x], device="cuda") for x in (512.0, 0.0, 1.0))
    want = s.expect(scale=512.0)
    s.run(grad_scale=scale, found_inf=fine)
    s.check(want)
    before = [t.clone() for t in s.all()]
    for g in s.g:
        g.fill_(float("inf"))
    kept = [g.clone() for g in s.g]
    s.run(grad_scale=scale, found_inf=bad)
    same = lambda a, b: torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
    now = s.all()
    g0 = len(s.p)
    for i, (a, b) in enumerate(zip(now, before)):
        if not g0 <= i < 2 * g0:
            assert same(a, b)
    assert all(torch.equal(a, b) for a, b in zip(s.g, kept)) and s.step.tolist() == [5, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_not_finite_stays_in_its_block(bits):
    """Its own moments with 32 bits, its block of 128 with 8; everything else is as without it."""
    a, b = (State(counts=[1000], param="fp32", bits=bits, seed=6) for _ in range(2))
    a.g[0][300], a.g[0][700] = float("nan"), float("inf")
    for s in (a, b):
        s.run()
    at = torch.zeros(1000, dtype=torch.bool, device="cuda")
    at[[300, 700]] = True
    assert torch.equal(a.p[0][~at], b.p[0][~at]) and not torch.isfinite(a.p[0][at]).any()
    if bits == 8:
        at[256:384] = at[640:768] = True
    for x, y in zip(a.moments(), b.moments()):
        assert torch.equal(x[0][~at], y[0][~at])
        assert not torch.isfinite(x[0][at]).any()


def test_codes_keep_the_mean():
    """Moments between two codes go to either with the probability that keeps the mean: over n values the mean is off by
    six standard deviations (at most half a code over the root of n each) at most."""
    n = 1 << 20
    s = State(counts=[n], param="fp32", bits=8, seed=7, steps=0)
    s.m[0].view(torch.uint8).zero_()
    s.v[0].view(torch.uint8).zero_()
    g = torch.empty(n, device="cuda").uniform_(0.5, 0.98, generator=torch.Generator(device="cuda").manual_seed(3))
    g.view(-1, 128)[:, 0] = 1.0
    s.g[0].copy_(g)
    s.run()
    for got, want in zip(s.moments(), ((1 - B1) * g.double(), (1 - B2) * g.double() ** 2)):
        code = want / want.view(-1, 128).amax(1).repeat_interleave(128) * 448
        deviation = (2.0 ** (torch.floor(torch.log2(code)) - 3) / 2 * (want / code)).square().sum().sqrt() / n
        assert abs(got[0].mean() - want.mean()) <= 6 * deviation


def test_a_slow_average_moves_in_8_bits():
    """v grows by 0.1 % of the way a step: with rounding to the nearest code it would never leave its own."""
    n = 128 * 512
    s = State(counts=[n], param="fp32", bits=8, seed=8, steps=1000)
    s.v[0].view(torch.uint8).fill_(0x70)  # 128
    s.vs[0].fill_(1.0 / 448)
    s.g[0].fill_((256.0 / 448) ** 0.5)
    s.g[0].view(-1, 128)[:, 0] = 1.0      # keeps the scale of every block where it is
    s.v[0].view(torch.uint8).view(-1, 128)[:, 0] = 0x7E
    for _ in range(200):
        s.run()
    want = 256.0 / 448 - 128.0 / 448 * B2 ** 200
    got = s.moments()[1][0].view(-1, 128)[:, 1:].mean().item()
    # each value wanders by at most the root of 200 steps' variances (p (1 - p) code^2, p = 0.001 * 128 / 16): 1.3 codes of 16 / 448
    assert abs(got - want) <= 6 * 1.3 * 16 / 448 / (n * 127 / 128) ** 0.5 + want * 2.0 ** -12


def test_same_bits_for_the_same_seed():
    a, b, c = (State(param="bf16", bits=8, seed=9) for _ in range(3))
    a.run(seed=5); b.run(seed=5); c.run(seed=6)
    bits = lambda s: torch.cat([t.view(torch.uint8) for t in s.m + s.v])
    assert torch.equal(bits(a), bits(b)) and not torch.equal(bits(a), bits(c))
    assert all(torch.equal(x, y) for x, y in zip(a.p, c.p))  # the step itself is taken with the values before they are rounded


@pytest.mark.parametrize("bits", [32, 8])
def test_on_a_stream_and_in_a_graph(bits):
    """Every replay is a further step; the rate is the one in memory."""
    lr = torch.full((1,), LR, device="cuda")
    a, b = (State(param="fp16", master=True, bits=bits, seed=10) for _ in range(2))
    rates = (LR, LR, 3 * LR, LR / 7)
    for r in rates:
        a.run(lr=torch.tensor([r], device="cuda"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.run(lr=lr)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(lr=lr)
    for r in rates[1:]:
        lr.fill_(r)
        graph.replay()
    view = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    assert all(torch.equal(view(x), view(y)) for x, y in zip(a.all(), b.all()))


def test_two_streams_at_once():
    a, b = State(param="fp32", bits=8, seed=11), State(param="fp32", bits=8, seed=12)
    wa, wb = a.expect(), b.expect()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for s, st in zip((a, b), streams):
        with torch.cuda.stream(st):
            s.run()
    torch.cuda.synchronize()
    a.check(wa)
    b.check(wb)


def test_autograd_notices():
    s = State(counts=[64], param="fp32")
    w = s.p[0].requires_grad_()
    loss = (w * w).sum()
    s.p = [w]
    s.run()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals():
    from fgms_b200 import backend
    def call(change):
        s = State(counts=[100, 200], param="fp32", bits=8)
        kw = dict(params=s.p, grads=s.g, exp_avgs=s.m, exp_avg_sqs=s.v, step=s.step, lr=LR, exp_avg_scales=s.ms, exp_avg_sq_scales=s.vs)
        change(kw)
        before = s.step.clone()
        try:
            backend.fgms_adamw_cuda(**kw)
        finally:
            assert torch.equal(before, s.step)
    put = lambda **kw: (lambda d: d.update(kw))
    at = lambda key, i, v: (lambda d: d[key].__setitem__(i, v(d[key][i])))
    for change, text in [
        (put(lr=-1.0), "lr"), (put(lr=float("nan")), "lr"), (put(beta1=1.0), "betas"), (put(beta2=-0.1), "betas"), (put(eps=0.0), "eps"),
        (put(weight_decay=-1.0), "weight_decay"), (put(seed=-1), "seed"), (put(seed=2 ** 32), "seed"),
        (lambda d: d["params"].pop(), "tensors, params"), (lambda d: d["exp_avg_scales"].pop(), "tensors, params"),
        (put(exp_avg_scales=None), "exp_avg_scales"),
        (at("grads", 1, lambda t: t[:50]), "must have 200 values"), (at("exp_avgs", 0, lambda t: t.float()), "dtype"),
        (at("exp_avg_scales", 1, lambda t: t[:1]), "must have 2 values"), (at("params", 0, lambda t: t.double()), "dtype"),
        (at("grads", 0, lambda t: t.cpu()), "must live on"), (at("params", 1, lambda t: torch.zeros(400, device="cuda")[::2]), "contiguous"),
        (lambda d: d["params"].__setitem__(1, torch.cat([d["params"][0], d["params"][0]])[:200]) or d["grads"].__setitem__(1, d["params"][1]), "overlaps"),
        (lambda d: [d[k].__setitem__(1, d[k][0]) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales")], "overlaps"),
        (put(step=torch.zeros(1, dtype=torch.int32, device="cuda")), "step"), (put(step=torch.zeros(2, dtype=torch.int64, device="cuda")), "step"),
        (put(grad_scale=torch.ones(2, device="cuda")), "grad_scale"), (put(found_inf=torch.zeros(1)), "found_inf"),
    ]:
        with pytest.raises(ValueError, match=text):
            call(change)
    with pytest.raises(TypeError):
        call(put(params=None))
    with pytest.raises(TypeError):
        call(at("grads", 0, lambda t: None))


# ---- the optimizer ------------------------------------------------------------------------------------------------------
def small_net(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 60), torch.nn.Linear(60, 30), torch.nn.Linear(30, 7, bias=False)).to("cuda", dtype)


def give_gradients(net, seed, scale=1.0, but=()):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for i, p in enumerate(net.parameters()):
        g = torch.randn(p.shape, generator=gen, device="cuda") * 0.01 * scale
        p.grad = None if i in but else g.to(p.dtype)


def test_optimizer_takes_pytorchs_steps():
    from fgms_b200 import optim
    a, b = small_net(), small_net()
    kw = dict(lr=1e-2, betas=(0.8, 0.99), eps=1e-7, weight_decay=0.1)
    mine, theirs = optim.AdamW(a.parameters(), **kw), torch.optim.AdamW(b.parameters(), **kw)
    for step in range(6):
        but = (1,) if step in (0, 3) else ()  # a parameter that joins later and misses a step
        give_gradients(a, step, but=but)
        give_gradients(b, step, but=but)
        mine.step()
        theirs.step()
    assert [int(mine.state[p]["step"][0]) for p in a.parameters()] == [6, 4, 6, 6, 6]
    for p, q in zip(a.parameters(), b.parameters()):
        # six updates of at most 3 lr each, every one off by 2^-20 on either side, and the values' own rounding
        assert ((p - q).abs() <= 2 * 6 * (3e-2 * 2.0 ** -20 + q.abs() * 2.0 ** -22)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded_state_goes_on_as_before(bits):
    from fgms_b200 import optim
    import io
    a, b = small_net(torch.bfloat16), small_net(torch.bfloat16)
    make = lambda net: optim.AdamW([{"params": list(net[0].parameters())}, {"params": list(net[1:].parameters()), "lr": 1e-2}], state_bits=bits)
    first, second = make(a), make(b)
    for step in range(3):
        give_gradients(a, step, but=(3,) if step == 0 else ())
        first.step()
    file = io.BytesIO()
    torch.save(first.state_dict(), file)
    file.seek(0)
    second.load_state_dict(torch.load(file))
    b.load_state_dict(a.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        assert {k: v.dtype for k, v in first.state[p].items()} == {k: v.dtype for k, v in second.state[q].items()}
    from fgms_b200 import backend
    for step in range(3, 5):
        give_gradients(a, step)
        give_gradients(b, step)
        first.step()
        launches = backend.launch_count()
        second.step()
        assert backend.launch_count() - launches == 3  # two groups, one of them with a parameter of its own count
    view = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and all(torch.equal(view(first.state[p][k]), view(second.state[q][k])) for k in first.state[p])


def test_small_updates_are_kept_by_masters():
    from fgms_b200 import optim
    for master in (True, False):
        w = torch.nn.Parameter(torch.ones(64, device="cuda", dtype=torch.bfloat16))
        opt = optim.AdamW([w], lr=1e-4, weight_decay=0.0, master=master)
        for _ in range(100):  # 100 steps of 1e-4: three steps of bf16 below 1 (2^-8 = 0.0039)
            w.grad = torch.ones_like(w)
            opt.step()
        assert (abs(1 - w.float().mean().item() - 0.01) <= 2.0 ** -9) if master else (w == 1).all()


def test_gradient_scaler():
    from fgms_b200 import optim
    a, b = small_net(torch.float16), small_net(torch.float16)
    scaled, plain = optim.AdamW(a.parameters()), optim.AdamW(b.parameters())
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0, growth_interval=1000)
    for step in range(4):
        give_gradients(b, step)
        for p, q in zip(a.parameters(), b.parameters()):
            p.grad = q.grad * 256.0
        if step == 2:
            next(a.parameters()).grad[0, 0] = float("inf")
        scaler.scale(torch.zeros((), device="cuda"))
        scaler.step(scaled)
        scaler.update()
        if step == 2:
            scaler.update(256.0)
        else:
            plain.step()
    assert [s["step"].tolist() for s in scaled.state.values()] == [[3, 0]] * 5
    # multiplying by 256 is exact unless a gradient overflows (none does); so are the steps
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_optimizer_refusals():
    from fgms_b200 import optim
    w = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=0.0), dict(weight_decay=-0.1), dict(state_bits=16), dict(seed=-1)):
        with pytest.raises(ValueError):
            optim.AdamW([w], **kw)
    with pytest.raises(ValueError, match="float32"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(8, device="cuda", dtype=torch.float64))])
    t = torch.nn.Parameter(torch.zeros((8, 4), device="cuda").T)
    t.grad = torch.zeros_like(t)
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([t]).step()
    e = torch.nn.Parameter(torch.zeros((8, 4), device="cuda"))
    e.grad = torch.zeros((8, 4), device="cuda").to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        optim.AdamW([e]).step()


def test_layers_of_experts_learn_in_one_step_each():
    """Products, their gradients and the update together, as a network uses them, against the same step in 64 bits."""
    from fgms_b200 import nn, optim
    torch.manual_seed(1)
    first, second = nn.GroupedLinear(64, 128, 4, dtype=torch.bfloat16), nn.GroupedLinear(128, 64, 4, dtype=torch.bfloat16)
    weights = [first.weight, second.weight]
    opt = optim.AdamW(weights, lr=1e-2, state_bits=8)
    kpos = torch.tensor([0, 50, 50, 90, 130], dtype=torch.int32, device="cuda")
    x, target = torch.randn((140, 64), device="cuda").bfloat16(), torch.randn((140, 64), device="cuda").bfloat16()
    before = [w.detach().double() for w in weights]
    hidden = first(x, kpos)
    loss = ((second(torch.relu(hidden), kpos) - target).float() ** 2).mean()
    loss.backward()
    wide = [w.clone().requires_grad_() for w in before]
    out = torch.zeros((140, 64), dtype=torch.float64, device="cuda")
    for g in range(4):
        s = slice(int(kpos[g]), int(kpos[g + 1]))
        out[s] = torch.relu(x[s].double() @ wide[0][g]) @ wide[1][g]
    ((out - target.double()) ** 2).mean().backward()
    for w, v in zip(weights, wide):
        # bf16 rounds at every stage: rows, their gradients (each 2^-9 of the value, and the hidden ones' signs near zero), the gradient itself
        assert (w.grad.double() - v.grad).norm() <= 8 * 2.0 ** -8 * v.grad.norm()
        assert not w.grad[1].any()
    grads = [w.grad.clone() for w in weights]
    opt.step()
    for w, b, g in zip(weights, before, grads):
        # the first step: lr * sign(gradient) where it is well above eps, the weight's rounding besides
        want = b * (1 - 1e-2 * 0.01) - 1e-2 * g.double() / (g.double().abs() + 1e-8)
        assert ((w.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-2 * 2.0 ** -18).all()


def one_operation_at_a_time(x, lot, floor):
    """Codes and scales in fp32, every operation rounded by itself: what the kernel computes two at a time."""
    n = x.numel()
    x, lot = blocks(x), blocks(lot)
    top = x.abs().amax(1, keepdim=True)
    scale = top * (1.0 / 448.0)
    u = (x.abs() * (torch.ones_like(scale) / scale)).clamp(max=448.0)
    normal = ((u.view(torch.int32) + (lot.int() << 4)) & -(1 << 20)).view(torch.float32)
    small = torch.floor(u * 512.0 + lot.float() * 2.0 ** -16)
    if floor:
        small = torch.where(u > 0, small.clamp(min=1.0), small)
    code = torch.copysign(torch.where(u >= 2.0 ** -6, normal, small * 2.0 ** -9), x)
    return code.view(-1)[:n].to(torch.float8_e4m3fn), scale.view(-1)


def mixed(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


@pytest.mark.parametrize("grad", ["fp32", "fp16", "bf16"])
def test_codes_are_the_same_bits_as_the_formulas_in_fp32(grad):
    """So that a step can be repeated, and checked, by anything that rounds as fp32 does."""
    s = State(counts=[128 * 4096, 1000, 77], param="fp32", grad=grad, bits=8, seed=13)
    s.g[0].view(-1, 128).mul_(torch.logspace(-3, 1, 4096, device="cuda").to(s.g[0].dtype)[:, None])
    for seed in (1, 2):
        want = []
        t = int(s.step[0]) + 1
        key = int(mixed(torch.tensor((t * 0x9E3779B9 & 0xFFFFFFFF) ^ seed)))
        f32 = lambda c, sc: (blocks(c.float()) * sc[:, None]).view(-1)[:c.numel()]
        for m, v, ms, vs, g in zip(s.m, s.v, s.ms, s.vs, s.g):
            g = g.float()
            m, v = f32(m, ms) * B1 + g * (1.0 - B1), f32(v, vs) * B2 + (g * g) * (1.0 - B2)
            h = mixed((torch.arange(g.numel(), device="cuda") * 0x9E3779B1 + key) & 0xFFFFFFFF)
            want.append((one_operation_at_a_time(m, h & 0xFFFF, False), one_operation_at_a_time(v, h >> 16, True)))
        s.run(seed=seed)
        for i, ((m, ms), (v, vs)) in enumerate(want):
            assert torch.equal(s.ms[i], ms) and torch.equal(s.vs[i], vs)
            assert torch.equal(s.m[i].float(), m.float()) and torch.equal(s.v[i].float(), v.float())


def test_values_beyond_32_bits():
    """A tensor of more than 2^31 values: the last ones take the step of the formula, those that an offset cut to 32 bits would meet keep to theirs."""
    from fgms_b200 import backend
    n = 2 ** 31 + 3000
    p = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-1000:] = 1.0
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros((n + 127) // 128, device="cuda") for _ in range(2))
    step = torch.zeros(2, dtype=torch.int32, device="cuda")
    backend.fgms_adamw_cuda([p], [g], [m], [v], step, 0.25, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    assert (p[-1000:] == 0.25).all() and (p[:5000] == 0.5).all() and (p[n // 2:n // 2 + 5000] == 0.5).all() and (p[-3000:-1000] == 0.5).all()
    assert ms[-1] > 0 and not ms[:-9].any() and vs[-1] > 0 and not vs[:-9].any()
    assert (m[-1000:].float() > 0).all() and (v[-1000:].float() > 0).all() and not m[-3000:-1000].float().any()


def test_optimizer_in_a_capture():
    """Refused where the state would be made anew by every replay: before the first step, and where a parameter parts from the others."""
    from fgms_b200 import optim
    a, b = small_net(), small_net()
    mine, other = optim.AdamW(a.parameters(), lr=1e-2), optim.AdamW(b.parameters(), lr=1e-2)
    give_gradients(a, 0)
    give_gradients(b, 0)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph, stream=side):
            mine.step()
    torch.cuda.synchronize()
    assert not any("exp_avg" in s for s in mine.state.values())
    mine.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mine.step()
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    kept = next(a.parameters()).grad
    next(a.parameters()).grad = None
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            mine.step()
    torch.cuda.synchronize()
    next(a.parameters()).grad = kept
    mine.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_of_different_types_in_a_group(bits):
    """float32 parameters have no master beside those that do; each takes the step that it takes alone."""
    from fgms_b200 import backend, optim
    make = lambda: [torch.nn.Parameter(torch.full((300,), 0.5, device="cuda", dtype=t)) for t in (torch.float32, torch.bfloat16, torch.float16)]
    together, alone = make(), make()
    opts = [optim.AdamW(together, lr=1e-2, state_bits=bits)], [optim.AdamW([p], lr=1e-2, state_bits=bits) for p in alone]
    for step in range(2):
        for params in (together, alone):
            for i, p in enumerate(params):
                p.grad = torch.linspace(-1, 1, 300, device="cuda").mul_(i + step + 1).to(p.dtype)
        launches = backend.launch_count()
        opts[0][0].step()
        assert backend.launch_count() - launches == 1
        for o in opts[1]:
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(together, alone))
    assert ["master" in opts[0][0].state[p] for p in together] == [False, True, True]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_whole_training_step_in_a_graph(bits):
    """Products, gradients and update captured together: replays take the steps that eager ones take, to the bit."""
    from fgms_b200 import nn, optim
    kpos = torch.tensor([0, 70, 70, 150, 200], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((210, 96), generator=gen, device="cuda").bfloat16()
    nets, opts = [], []
    for _ in range(2):
        torch.manual_seed(2)
        nets.append(torch.nn.ModuleList([nn.GroupedLinear(96, 256, 4, dtype=torch.bfloat16), nn.GroupedLinear(256, 96, 4, dtype=torch.bfloat16)]))
        opts.append(optim.AdamW(nets[-1].parameters(), lr=1e-2, state_bits=bits))

    def step(i):
        out = nets[i][1](torch.relu(nets[i][0](x, kpos)), kpos)
        ((out - x).float() ** 2).mean().backward()
        opts[i].step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(1)
        opts[1].zero_grad(set_to_none=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opts[1].zero_grad(set_to_none=True)
        step(1)
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        opts[0].zero_grad(set_to_none=True)
        step(0)
    assert opts[1].state[nets[1][0].weight]["step"].tolist() == [4, 0]
    assert all(torch.equal(p, q) for p, q in zip(nets[0].parameters(), nets[1].parameters()))


@pytest.mark.parametrize("size", [1e-13, 1e-15, 1e-17, 1e-19, 1e-20])
def test_a_tiny_second_moment_stays_above_zero_in_8_bits(size):
    """A block of gradients so small that their squares are near fp32's smallest numbers, then none: the update is that of the moments, not m divided
    by eps.  A value of v is off by a code at most, an eighth of it or 2^-135, and by fp32's subnormal steps before that.

    The second step is exactly 0.9 * 0.1 / 0.19 / sqrt(0.999 * 0.001 / 0.001999) = 0.670 of the rate; with m off by an eighth upwards and v downwards (where it is
    off by more it is larger) at most 0.670 * 1.125 / sqrt(0.875) = 0.81 of it."""
    from fgms_b200 import backend
    lr, n = 0.5, 300
    p = torch.ones(n, device="cuda")
    g = torch.full((n,), size, device="cuda")
    g[::3] *= -0.5
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros(3, device="cuda") for _ in range(2))
    step = torch.zeros(2, dtype=torch.int32, device="cuda")
    call = lambda: backend.fgms_adamw_cuda([p], [g], [m], [v], step, lr, B1, B2, 1e-30, 0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    want = (1 - B2) * g.double() ** 2
    call()
    got = held(v, vs)
    assert (got > 0).all()
    assert ((got - want).abs() <= (want / 8).clamp(min=2.0 ** -135) * (1 + 2.0 ** -20) + 2.0 ** -147).all()
    before = p.clone()
    g.zero_()
    call()
    assert (held(v, vs) > 0).all()
    assert ((p - before).abs() <= 0.82 * lr).all()


def test_a_block_of_zeros_is_held_as_zeros():
    s = State(counts=[300], param="fp32", bits=8, seed=14, steps=0)
    for t in (s.m[0].view(torch.uint8), s.v[0].view(torch.uint8), s.ms[0], s.vs[0]):
        t.zero_()
    s.g[0][:128] = 0
    s.run()
    assert not s.m[0].float()[:128].any() and not s.v[0].float()[:128].any() and s.ms[0][0] == 0 and s.vs[0][0] == 0
    assert s.vs[0][1] > 0


@pytest.mark.parametrize("keep", [8, 64])
@pytest.mark.parametrize("bits", [32, 8])
def test_with_sms_kept_free(bits, keep):
    """Steps behind one another, of several launches each: the same as with all SMs, to the bit."""
    from fgms_b200 import _lib
    kept, free = (State(counts=[(i * 37) % 300 for i in range(450)] + [100003], param="fp16", master=True, bits=bits, seed=15) for _ in range(2))
    for _ in range(3):
        free.run()
    assert _lib.lib.fgms_b200_set_reserved_sms(keep) == _lib.OK
    try:
        for _ in range(3):
            kept.run()
    finally:
        _lib.lib.fgms_b200_set_reserved_sms(0)
    view = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    assert all(torch.equal(view(a), view(b)) for a, b in zip(kept.all(), free.all()))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_whose_square_is_not_finite(bits):
    """The step itself is that of the formula (an infinite denominator for the value, everything else as without it).  Its second moment is infinite from then on,
    with 8 bits that of its block NaN; first moments stay finite."""
    a, b = (State(counts=[1000], param="fp32", bits=bits, seed=16) for _ in range(2))
    a.g[0][300] = 1e20
    before = a.p[0][300].item()
    for s in (a, b):
        s.run()
    at = torch.zeros(1000, dtype=torch.bool, device="cuda")
    at[300] = True
    assert torch.equal(a.p[0][~at], b.p[0][~at])
    assert abs(a.p[0][300].item() - before * (1 - LR * DECAY)) <= abs(before) * 2.0 ** -22
    (m,), (v,) = a.moments()
    assert torch.isfinite(m).all()
    if bits == 8:
        at[256:384] = True
        assert torch.isnan(v[at]).all()
    else:
        assert torch.isinf(v[at]).all()
    assert torch.equal(v[~at], b.moments()[1][0][~at])
