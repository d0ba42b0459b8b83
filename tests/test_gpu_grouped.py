"""Products of ragged groups of rows against the definition in 64 bits.

A computed value may be off by the rounding to its type, half a step, and by the fp32 sum before it: n products added in any order, with
every addition off by a step (2^-23) of the partial sum at most, which no partial sum of the absolute values exceeds.  (n + 1: the products
of fp32 values are rounded as well; those of 16-bit values are exact.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def kpos_of(sizes, start=0):
    k = [start]
    for n in sizes:
        k.append(k[-1] + n)
    return torch.tensor(k, dtype=torch.int32, device="cuda")


def near(got, exact, magnitude, n):
    """Every value of `got` within what its type and a sum of n products allow."""
    t = got.dtype
    smallest = torch.finfo(t).smallest_normal * torch.finfo(t).eps  # step of the subnormal numbers
    allowed = exact.abs() * (torch.finfo(t).eps / 2) + magnitude * ((n + 1) * 2.0 ** -23) * (1 + torch.finfo(t).eps) + smallest
    off = (got.double() - exact).abs()
    assert torch.isfinite(got).all()
    worst = (off - allowed).max().item() if off.numel() else 0.0
    assert worst <= 0, f"off by {worst} more than allowed"


class Layer:
    """Inputs of a layer; rows of no group hold NaN, outputs 7."""

    def __init__(self, dtype, sizes, c_in, c_out, start=0, rest=0, seed=0, fill=float("nan")):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        t = TYPES[dtype]
        self.sizes, self.rows, self.start = list(sizes), start + sum(sizes) + rest, start
        self.kpos = kpos_of(sizes, start)
        normal = lambda *s: torch.randn(s, generator=gen, device="cuda")
        self.x, self.g = normal(self.rows, c_in), normal(self.rows, c_out)
        inside = torch.zeros(self.rows, dtype=torch.bool, device="cuda")
        inside[start:start + sum(sizes)] = True
        self.inside = inside
        for v in (self.x, self.g):
            v[~inside] = fill
        self.x, self.g = self.x.to(t), self.g.to(t)
        self.w = (normal(len(sizes), c_in, c_out) * c_in ** -0.5).to(t)

    def each(self):
        at = self.start
        for g, n in enumerate(self.sizes):
            yield g, slice(at, at + n)
            at += n

    def exact(self, which):
        """(values, the same of the absolute values, length of the sums)"""
        out = []
        for f in (lambda v: v.double(), lambda v: v.double().abs()):
            x, g, w = f(self.x), f(self.g), f(self.w)
            if which == "wgrad":
                r = torch.zeros_like(w)
                for i, s in self.each():
                    r[i] = x[s].T @ g[s]
            else:
                r = torch.zeros_like(g if which == "fwd" else x)
                for i, s in self.each():
                    r[s] = x[s] @ w[i] if which == "fwd" else g[s] @ w[i].T
            out.append(r)
        n = {"fwd": self.w.size(1), "dgrad": self.w.size(2), "wgrad": max(self.sizes, default=0)}[which]
        return out[0], out[1], n

    def run(self, which, zero_rest=False):
        from fgms_b200 import backend
        if which == "wgrad":
            out = torch.full_like(self.w, 7)
            backend.fgms_grouped_wgrad_cuda(self.x, self.g, out, self.kpos)
        elif which == "fwd":
            out = torch.full_like(self.g, 7)
            backend.fgms_grouped_fwd_cuda(self.x, self.w, out, self.kpos, zero_rest)
        else:
            out = torch.full_like(self.x, 7)
            backend.fgms_grouped_dgrad_cuda(self.g, self.w, out, self.kpos, zero_rest)
        return out

    def check(self, which, zero_rest=False):
        got = self.run(which, zero_rest)
        exact, magnitude, n = self.exact(which)
        if which == "wgrad":
            near(got, exact, magnitude, n)
        else:
            near(got[self.inside], exact[self.inside], magnitude[self.inside], n)
            assert (got[~self.inside] == (0 if zero_rest else 7)).all()
        return got


PASSES = ("fwd", "dgrad", "wgrad")
# one row, one channel, widths around the tiles' edges and off every boundary, empty groups, one group alone, many small ones
SHAPES = [
    ([1], 1, 1), ([1], 8, 8), ([3, 0, 1], 16, 24), ([5], 7, 9), ([0, 0], 64, 64), ([130, 0, 64, 1, 127], 72, 136),
    ([128, 256], 128, 256), ([257, 1, 0, 300], 200, 264), ([63, 65, 129], 65, 127), ([17] * 40, 96, 64), ([0, 513, 0], 320, 520),
    ([40, 2, 9], 1000, 8), ([40, 2, 9], 8, 1000), ([700, 900], 512, 768),
]


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sizes,c_in,c_out", SHAPES, ids=[f"{len(s)}g{sum(s)}r_{a}x{b}" for s, a, b in SHAPES])
def test_against_the_definition(sizes, c_in, c_out, dtype, which):
    from fgms_b200 import backend
    backend.device_status()
    Layer(dtype, sizes, c_in, c_out, seed=len(sizes) + c_in).check(which)
    assert backend.device_status() == 0


# few tiles with a long contraction, which several CTAs share: channels for the products of rows, rows for the weight gradient
LONG = [([1], 4096, 4096), ([20], 4000, 200), ([1, 0, 6], 2056, 136), ([33, 60], 2560, 72), ([1000], 4096, 128), ([5], 200, 4096), ([30, 9], 136, 3000),
        ([3000], 256, 256), ([5000, 3, 0], 128, 264), ([8001], 504, 512), ([2047, 1], 24, 40), ([9000, 4000], 64, 64)]


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("sizes,c_in,c_out", LONG, ids=[f"{len(s)}g{sum(s)}r_{a}x{b}" for s, a, b in LONG])
def test_long_contractions(sizes, c_in, c_out, dtype, which):
    from fgms_b200 import backend
    backend.device_status()
    layer = Layer(dtype, sizes, c_in, c_out, start=3, rest=40, seed=len(sizes) + c_in)
    first = layer.check(which)
    assert torch.equal(first, layer.run(which))
    if which != "wgrad":
        layer.check(which, zero_rest=True)
    assert backend.device_status() == 0


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("c_in,c_out", [(64, 128), (50, 33)])
def test_rows_of_no_group(dtype, which, c_in, c_out):
    """Not read (they hold NaN) and left as they were, or cleared."""
    layer = Layer(dtype, [70, 0, 131, 5], c_in, c_out, start=9, rest=77, seed=3)
    layer.check(which)
    if which != "wgrad":
        layer.check(which, zero_rest=True)


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinities_and_nan_stay_in_their_group(dtype, which):
    """A group whose weights or rows are not finite leaves the groups beside it in the same tiles alone."""
    layer = Layer(dtype, [20, 30, 25], 72, 88, seed=5)
    want = layer.run(which)
    layer.x[20:50] = float("inf")
    layer.g[20:50] = float("nan")
    layer.w[1] = float("nan")
    got = layer.run(which)
    if which == "wgrad":
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.isnan(got[1]).any()
    else:
        assert torch.equal(got[:20], want[:20]) and torch.equal(got[50:], want[50:]) and torch.isnan(got[20:50]).any()


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_same_bits_on_every_run(dtype, which):
    layer = Layer(dtype, [300, 17, 0, 450], 256, 384, seed=6)
    first = layer.run(which)
    for _ in range(3):
        assert torch.equal(first, layer.run(which))


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_views_that_start_off_a_boundary(dtype, which, shift):
    layer = Layer(dtype, [33, 100], 64, 72, seed=7)
    def moved(v):
        flat = torch.empty(v.numel() + shift, dtype=v.dtype, device="cuda")
        out = flat[shift:].view(v.shape)
        out.copy_(v)
        return out
    layer.x, layer.g, layer.w = moved(layer.x), moved(layer.g), moved(layer.w)
    layer.check(which)


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("bad,good,count", [
    ([0, 60, 40, 100], [0, 60, 60, 100], 1),          # an entry out of order: the group is empty
    ([-5, 10, 20, 30], [0, 10, 20, 30], 1),
    ([0, 50, 4000, 100], [0, 50, 100, 100], 1),
    ([0, 2**31 - 1, -2**31, 7], [0, 100, 100, 100], 3),
])
def test_bad_kpos_is_counted_and_stays_inside(dtype, which, bad, good, count):
    from fgms_b200 import backend
    layer = Layer(dtype, [100], 64, 40, seed=8)
    layer.w = layer.w.expand(3, -1, -1).contiguous()
    layer.kpos = torch.tensor(good, dtype=torch.int32, device="cuda")
    want = layer.run(which)
    backend.device_status()
    layer.kpos = torch.tensor(bad, dtype=torch.int32, device="cuda")
    got = layer.run(which)
    assert torch.equal(got, want)
    assert backend.device_status() == count


def test_no_rows_at_all():
    from fgms_b200 import backend
    layer = Layer("bf16", [0, 0, 0], 64, 64)
    assert layer.run("fwd").shape == (0, 64) and layer.run("dgrad").shape == (0, 64)
    assert (layer.run("wgrad") == 0).all()
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_most_groups(dtype):
    sizes = [(i * 7) % 5 for i in range(1024)]
    for which in PASSES:
        Layer(dtype, sizes, 32, 40, rest=3, seed=9).check(which)


@pytest.mark.parametrize("which", PASSES)
def test_long_rows_and_many(which):
    """The contraction over thousands of channels or rows, tiles by the thousand."""
    Layer("bf16", [2000, 3, 2500, 500], 1536, 2304, rest=11, seed=10).check(which)


def test_offsets_beyond_32_bits():
    """A weight tensor of more than 2^32 bytes and 2^31 values: the last matrix is the one that is multiplied with."""
    groups, c = 520, 2048
    from fgms_b200 import backend
    w = torch.zeros((groups, c, c), dtype=torch.float16, device="cuda")
    w[-1] = torch.eye(c, device="cuda", dtype=torch.float16) * 3
    x = torch.randn((5, c), device="cuda").half()
    kpos = kpos_of([0] * (groups - 1) + [5])
    out = torch.empty_like(x)
    backend.fgms_grouped_fwd_cuda(x, w, out, kpos)
    assert torch.equal(out, x * 3)
    backend.fgms_grouped_dgrad_cuda(x, w, out, kpos)
    assert torch.equal(out, x * 3)
    backend.fgms_grouped_wgrad_cuda(x, x, w, kpos)
    assert not w[:-1].any()
    near(w[-1], x.double().T @ x.double(), x.double().abs().T @ x.double().abs(), 5)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_by_autograd(dtype):
    from fgms_b200 import nn
    layer = Layer(dtype, [90, 0, 140, 3], 80, 96, start=4, rest=21, seed=11)
    x, w = layer.x.clone().requires_grad_(), layer.w.clone().requires_grad_()
    out = nn.grouped_linear(x, w, layer.kpos)
    exact, magnitude, n = layer.exact("fwd")
    near(out.detach(), exact, magnitude, n)
    gx, gw = torch.autograd.grad(out, (x, w), layer.g)
    near(gx, *layer.exact("dgrad"))
    near(gw, *layer.exact("wgrad"))
    # one of the two alone, and an output gradient that is a broadcast
    (only,) = torch.autograd.grad(nn.grouped_linear(x, layer.w, layer.kpos), (x,), layer.g)
    assert torch.equal(only, gx)
    (only,) = torch.autograd.grad(nn.grouped_linear(layer.x, w, layer.kpos), (w,), layer.g)
    assert torch.equal(only, gw)
    layer.g = torch.ones((), dtype=layer.g.dtype, device="cuda").expand_as(layer.g)
    gx, gw = torch.autograd.grad(nn.grouped_linear(x, w, layer.kpos).sum(), (x, w))
    near(gx, *layer.exact("dgrad"))
    near(gw, *layer.exact("wgrad"))


def test_gradients_against_differences():
    """fp32: (f(v + h d) - f(v - h d)) / 2h of a product is exact but for rounding, as it is linear in either input."""
    from fgms_b200 import nn
    layer = Layer("fp32", [37, 0, 50], 24, 40, seed=12)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w = layer.x.clone().requires_grad_(), layer.w.clone().requires_grad_()
    value = lambda x, w: (nn.grouped_linear(x, w, layer.kpos).double() * layer.g.double()).sum()
    value(x, w).backward()
    for v, other, grad in ((layer.x, 0, x.grad), (layer.w, 1, w.grad)):
        d = torch.randn(v.shape, generator=gen, device="cuda")
        h = 0.5
        hi, lo = v + h * d, v - h * d
        pair = (lambda a: value(a, layer.w)) if other == 0 else (lambda a: value(layer.x, a))
        slope = (pair(hi) - pair(lo)) / (2 * h)
        # both sides: every output off by (c_in + 1) 2^-23 of the absolute products, inputs rounded once more
        big = Layer.__new__(Layer)
        big.__dict__.update(layer.__dict__)
        big.x, big.w = layer.x.abs() + (h * d.abs() if other == 0 else 0), layer.w.abs() + (h * d.abs() if other == 1 else 0)
        size = (big.exact("fwd")[1] * layer.g.double().abs()).sum()
        assert abs(slope - (grad.double() * d.double()).sum()) <= 4 * 60 * 2.0 ** -23 * size


def test_module_and_its_parameters():
    from fgms_b200 import nn
    net = nn.GroupedLinear(48, 64, 5, dtype=torch.bfloat16)
    assert net.weight.shape == (5, 48, 64) and net.weight.abs().max() <= 48 ** -0.5 * (1 + 2.0 ** -8)
    x = torch.randn((30, 48), device="cuda").bfloat16()
    kpos = kpos_of([10, 0, 5, 5, 10])
    assert torch.equal(net(x, kpos), nn.grouped_linear(x, net.weight, kpos))


def test_transposed_inputs_of_autograd():
    """Inputs that are no contiguous tensors are copied, as the layers of a map do."""
    from fgms_b200 import nn
    layer = Layer("fp16", [64, 10], 40, 56, seed=13)
    xt, wt = layer.x.T.contiguous().T, layer.w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(nn.grouped_linear(xt, wt, layer.kpos), nn.grouped_linear(layer.x, layer.w, layer.kpos))


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_on_a_stream_and_in_a_graph(dtype, which):
    layer = Layer(dtype, [200, 31, 0, 90], 128, 192, rest=9, seed=14, fill=0.0)
    want = layer.run(which)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.run(which)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.run(which)
    graph.replay()
    assert torch.equal(got, want)
    # other rows and other groups in the same buffers
    layer.x.mul_(2)
    layer.g.mul_(0.5)
    layer.kpos.copy_(kpos_of([100, 100, 100, 10]))
    want = layer.run(which)
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_two_streams_at_once(dtype):
    layers = [Layer(dtype, [400, 100, 300], 256, 320, seed=s) for s in (15, 16)]
    want = [[l.run(w) for w in PASSES] for l in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (l, st) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(st):
                got[i] = [l.run(w) for w in PASSES]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_a_training_step_in_a_graph_beside_an_eager_one():
    from fgms_b200 import nn
    layer = Layer("bf16", [100, 0, 60], 64, 128, seed=17)
    x, w = layer.x.clone().requires_grad_(), layer.w.clone().requires_grad_()
    step = lambda: torch.autograd.grad(nn.grouped_linear(x, w, layer.kpos), (x, w), layer.g)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_refusals():
    from fgms_b200 import backend, nn
    x = torch.zeros((10, 16), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros((3, 16, 24), device="cuda", dtype=torch.bfloat16)
    out = torch.zeros((10, 24), device="cuda", dtype=torch.bfloat16)
    kpos = kpos_of([5, 0, 5])
    fwd = backend.fgms_grouped_fwd_cuda
    for args, text in [
        ((x, w.half(), out, kpos), "dtype"), ((x.half(), w, out, kpos), "dtype"), ((x, w, out.float(), kpos), "dtype"),
        ((x.double(), w.double(), out.double(), kpos), "unsupported feature dtype"),
        ((x, w, out, kpos.long()), "int32"), ((x, w, out, kpos.cpu()), "must live on"), ((x, w, out, kpos[:3]), "one entry more"),
        ((x, w, out, kpos.view(2, 2)), "one entry more"), ((x[:, :8], w, out, kpos), "contiguous"), ((x, w, out[:5], kpos), "differ in rows"),
        ((x[:, :8].contiguous(), w, out, kpos), "channels"), ((x, w, out[:, :8].contiguous(), kpos), "channels"),
        ((x, w[0], out, kpos), "dimensions"), ((x[0], w, out, kpos), "dimensions"), ((x, w, x.new_zeros((10, 24)).T.contiguous().T, kpos), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            fwd(*args)
    with pytest.raises(ValueError, match="overlaps"):
        both = torch.zeros((3, 16, 16), device="cuda")
        fwd(both.view(48, 16)[:10], both, both.view(48, 16)[10:20], kpos)
    with pytest.raises(ValueError, match="differ in rows"):
        backend.fgms_grouped_wgrad_cuda(x[:9], out, w, kpos)
    with pytest.raises(ValueError, match="one entry more"):
        nn.grouped_linear(x, w, kpos[:2])


def test_a_second_derivative_is_refused_when_it_is_taken():
    from fgms_b200 import nn
    layer = Layer("fp32", [20, 30], 16, 24, seed=18)
    x, w = layer.x.clone().requires_grad_(), layer.w.clone().requires_grad_()
    gx, gw = torch.autograd.grad((nn.grouped_linear(x, w, layer.kpos) ** 2).sum(), (x, w), create_graph=True)
    plain = torch.autograd.grad((nn.grouped_linear(x, w, layer.kpos) ** 2).sum(), (x, w))
    assert torch.equal(gx, plain[0]) and torch.equal(gw, plain[1])
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        (gx.sum() + gw.sum()).backward()
    (only,) = torch.autograd.grad((nn.grouped_linear(x, layer.w, layer.kpos) ** 2).sum(), (x,), create_graph=True)
    assert torch.equal(only, plain[0])


def test_autograd_notices_that_an_output_was_written():
    from fgms_b200 import backend
    layer = Layer("fp32", [20, 30], 16, 24, seed=19)
    out = torch.ones_like(layer.g, requires_grad=True)
    loss = (out * out).sum()
    with torch.no_grad():
        backend.fgms_grouped_fwd_cuda(layer.x, layer.w, out, layer.kpos)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("keep", [8, 64])
def test_with_sms_kept_free(which, keep):
    from fgms_b200 import _lib
    assert _lib.lib.fgms_b200_set_reserved_sms(keep) == _lib.OK
    try:
        for dtype, sizes, c_in, c_out in (("bf16", [300, 0, 700], 256, 520), ("bf16", [3], 4096, 136), ("fp32", [300, 0, 70], 100, 130)):
            Layer(dtype, sizes, c_in, c_out, seed=20).check(which)
    finally:
        _lib.lib.fgms_b200_set_reserved_sms(0)


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("c_in,c_out", [(8, 70000), (70000, 8), (1, 40001)])
def test_very_wide(dtype, which, c_in, c_out):
    Layer(dtype, [3, 0, 14], c_in, c_out, seed=21).check(which)


def test_rows_beyond_32_bits():
    """More than 2^31 values in the rows: the last ones are the ones that are multiplied."""
    from fgms_b200 import backend
    rows, c = (1 << 20) + 77, 2056
    x = torch.zeros((rows, c), dtype=torch.float16, device="cuda")
    x[-70:] = torch.randn((70, c), device="cuda").half()
    w = (torch.randn((2, c, 64), device="cuda") * c ** -0.5).half()
    kpos = kpos_of([rows - 50, 50])
    out = torch.empty((rows, 64), dtype=torch.float16, device="cuda")
    backend.fgms_grouped_fwd_cuda(x, w, out, kpos)
    for s, i in ((slice(-70, -50), 0), (slice(-50, None), 1)):
        near(out[s], x[s].double() @ w[i].double(), x[s].double().abs() @ w[i].double().abs(), c)
    assert not out[:-70].any()
    dw = torch.empty_like(w)
    out.fill_(1)
    backend.fgms_grouped_wgrad_cuda(x, out, dw, kpos)
    for s, i in ((slice(-70, -50), 0), (slice(-50, None), 1)):
        want = x[s].double().sum(0)[:, None].expand(-1, 64)
        near(dw[i], want, x[s].double().abs().sum(0)[:, None].expand(-1, 64), 70)
    back = torch.empty_like(x)
    out.zero_()
    out[-50:] = 1
    backend.fgms_grouped_dgrad_cuda(out, w, back, kpos)
    near(back[-50:], w[1].double().sum(1).expand(50, -1), w[1].double().abs().sum(1).expand(50, -1), 64)
    assert not back[:-50].any()


@pytest.mark.parametrize("which", PASSES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("sizes,c_in,c_out,shift", [([300, 0, 700], 1001, 1003, 0), ([900, 40, 1500], 512, 517, 0), ([2100, 300], 257, 1024, 0),
                                                    ([400, 600, 128], 1024, 768, 1), ([400, 600, 128], 1024, 768, 4), ([30000], 65, 131, 0)])
def test_rows_that_are_copied_to_boundaries(sizes, c_in, c_out, shift, dtype, which):
    """Widths that are no multiples of 8 and views off a boundary, in calls that are large enough for copies to pay."""
    from fgms_b200 import _lib, backend
    layer = Layer(dtype, sizes, c_in, c_out, start=5, rest=30, seed=22)
    if shift:
        def moved(v):
            flat = torch.empty(v.numel() + shift, dtype=v.dtype, device="cuda")
            flat[shift:].view(v.shape).copy_(v)
            return flat[shift:].view(v.shape)
        layer.x, layer.g, layer.w = moved(layer.x), moved(layer.g), moved(layer.w)
    a, b, d = {"fwd": (layer.x, layer.w, layer.g), "dgrad": (layer.g, layer.w, layer.x), "wgrad": (layer.x, layer.g, layer.w)}[which]
    copied = _lib.lib.fgms_b200_grouped_workspace_bytes(PASSES.index(which), a.data_ptr(), b.data_ptr(), d.data_ptr(), layer.rows, c_in, c_out,
                                                        len(sizes), {"fp16": _lib.DTYPE_F16, "bf16": _lib.DTYPE_BF16}[dtype])
    assert copied > 0
    fallbacks, launches = backend.fallback_count(), backend.launch_count()
    first = layer.check(which)
    assert backend.fallback_count() == fallbacks and backend.launch_count() - launches >= 2
    assert torch.equal(first, layer.run(which))
    if which != "wgrad":
        layer.check(which, zero_rest=True)
    backend.device_status()
    layer.kpos[1] = layer.rows + 7        # one entry out of range, and the ones behind it out of order
    out = layer.run(which)
    assert backend.device_status() == len(sizes)
    if which != "wgrad":  # all rows from the first on are the first group's
        rows = slice(5, 5 + sum(sizes))
        x, w = (layer.x, layer.w[0]) if which == "fwd" else (layer.g, layer.w[0].T)
        near(out[rows], x[rows].double() @ w.double(), x[rows].double().abs() @ w.double().abs(), w.size(0))
        assert (out[:5] == 7).all()


def test_copied_rows_in_a_graph():
    """The workspace is the graph's own."""
    layers = [Layer("bf16", [500, 700], 513, 771, seed=s, fill=0.0) for s in (23, 24)]
    want = [[l.run(w) for w in PASSES] for l in layers]
    graphs, got = [], []
    for l in layers:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append([l.run(w) for w in PASSES])
    for _ in range(2):
        for g in graphs:
            g.replay()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_workspace_is_checked():
    from fgms_b200 import _lib
    layer = Layer("bf16", [500, 700], 513, 771, seed=25)
    out = torch.empty_like(layer.g)
    need = _lib.lib.fgms_b200_grouped_workspace_bytes(0, layer.x.data_ptr(), layer.w.data_ptr(), out.data_ptr(), layer.rows, 513, 771, 2, _lib.DTYPE_BF16)
    ws = torch.empty(need + 512, dtype=torch.uint8, device="cuda")
    call = lambda at, size: _lib.lib.fgms_b200_grouped_fwd(layer.x.data_ptr(), layer.w.data_ptr(), out.data_ptr(), layer.kpos.data_ptr(), layer.rows, 513, 771, 2,
                                                           _lib.DTYPE_BF16, 0, at, size, torch.cuda.current_stream().cuda_stream)
    assert call(ws.data_ptr(), need - 1) == _lib.ERR_WORKSPACE and call(ws.data_ptr() + 16, need) == _lib.ERR_WORKSPACE
    assert call(layer.w.data_ptr() // 256 * 256, need) == _lib.ERR_WORKSPACE
    exact, magnitude, n = layer.exact("fwd")
    for at, size in ((ws.data_ptr(), need), (None, 0)):  # without one: the CUDA cores
        out.zero_()
        assert call(at, size) == _lib.OK
        near(out, exact, magnitude, n)


def test_a_group_of_many_million_rows():
    """A tile whose stages take longer than any single wait is no wait that ran out (the other groups keep it from being shared by several CTAs)."""
    from fgms_b200 import backend
    rows, groups = 500_000_000, 200
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    g = torch.ones((rows, 8), dtype=torch.bfloat16, device="cuda")
    x[::250_000_000] = 1
    x[-1] = 2
    dw = torch.empty((groups, 8, 8), dtype=torch.bfloat16, device="cuda")
    kpos = torch.full((groups + 1,), rows, dtype=torch.int32, device="cuda")
    kpos[0] = 0
    backend.device_status()
    backend.fgms_grouped_wgrad_cuda(x, g, dw, kpos)
    assert backend.device_status() == 0
    assert (dw[0] == 4).all() and not dw[1:].any()


def test_ragged_groups_behind_many_million_rows():
    """The rows behind a group's last one are cleared by a warp that passes over tiles without such rows: its wait lasts as long as all of those
    may take.  Whichever tiles the first group's CTA gets next, their groups end inside a stage."""
    from fgms_b200 import backend
    first, groups = 499_999_984, 200  # a multiple of 16: nothing to clear
    rows = first + 5 * (groups - 1)
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    g = torch.ones((rows, 8), dtype=torch.bfloat16, device="cuda")
    x[::250_000_000] = 1
    x[first:] = torch.arange(1, groups, device="cuda").bfloat16().repeat_interleave(5)[:, None] * 2.0 ** -8
    dw = torch.empty((groups, 8, 8), dtype=torch.bfloat16, device="cuda")
    kpos = kpos_of([first] + [5] * (groups - 1))
    backend.device_status()
    backend.fgms_grouped_wgrad_cuda(x, g, dw, kpos)
    assert backend.device_status() == 0
    assert (dw[0] == 2).all()
    want = 5 * torch.arange(1, groups, device="cuda").double() * 2.0 ** -8  # exact in fp32, rounded once
    assert torch.equal(dw[1:], want.bfloat16()[:, None, None].expand(-1, 8, 8))


_ORDER = """
import sys, hashlib, torch
from fgms_b200 import backend
gen = torch.Generator(device="cuda").manual_seed(1)
def call(c_in, c_out):
    w = torch.randn((1, c_in, c_out), generator=gen, device="cuda").bfloat16()
    x = torch.randn((1, c_in), generator=gen, device="cuda").bfloat16()
    x[0, 0], x[0, -1] = 2.0 ** 20, -2.0 ** 20  # so large that the order of the sums shows in every value
    w[0, -1] = w[0, 0]
    out = torch.empty((1, c_out), device="cuda", dtype=torch.bfloat16)
    backend.fgms_grouped_fwd_cuda(x, w, out, torch.tensor([0, 1], device="cuda", dtype=torch.int32))
    return hashlib.sha256(out.view(torch.int16).cpu().numpy().tobytes()).hexdigest()
if sys.argv[1] == "behind":
    call(768, 768)
    gen.manual_seed(1)
print(call(4096, 1024))
"""


def test_same_bits_whichever_call_came_first():
    """How a contraction is shared out, and so the order of its sums, does not depend on the calls before: each in a process of its own."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    bits = []
    for order in ("alone", "behind"):
        run = subprocess.run([sys.executable, "-c", _ORDER, order], capture_output=True, text=True, cwd=root, timeout=300)
        assert run.returncode == 0, run.stderr
        bits.append(run.stdout.strip())
    assert bits[0] == bits[1] and len(bits[0]) == 64


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_cleared_for_the_other_cta_of_a_pair(dtype):
    """Weight gradient of groups that all end inside a stage, tile after tile by pairs of CTAs: each clears its part of what the even one's MMAs read.
    What lies behind a group's last row is the next group's, a thousand times as large; behind the last group NaN."""
    layer = Layer(dtype, [301 + 38 * i for i in range(16)], 1024, 1024, rest=40, seed=26)
    for i, s in layer.each():
        layer.x[s] *= 2.0 ** (10 * (i % 2) - 5)
    first = layer.check("wgrad")
    for _ in range(10):
        assert torch.equal(first, layer.run("wgrad"))


@pytest.mark.parametrize("keep", [8, 64])
def test_copied_rows_with_sms_kept_free(keep):
    from fgms_b200 import _lib, backend
    layer = Layer("bf16", [300, 0, 700], 1001, 1003, start=5, rest=30, seed=27)
    assert _lib.lib.fgms_b200_set_reserved_sms(keep) == _lib.OK
    try:
        for which in PASSES:
            launches = backend.launch_count()
            layer.check(which)
            assert backend.launch_count() - launches >= 2
            if which != "wgrad":
                layer.check(which, zero_rest=True)
    finally:
        _lib.lib.fgms_b200_set_reserved_sms(0)
