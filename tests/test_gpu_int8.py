"""Products in 8 bits against the definition in 64 bits.  The sum is an exact integer; what may be off is its rounding to fp32 and two
multiplications, 2^-24 each, and the rounding to the output's type."""
import pytest
import torch

from tests.layers_ref import near, tiny

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def kpos_of(sizes, start=0):
    k = [start]
    for n in sizes:
        k.append(k[-1] + n)
    return torch.tensor(k, dtype=torch.int32, device="cuda")


class Layer:
    """Codes over the whole range, -128 too; scales of rows of no group are NaN; rows `room` bytes apart beyond a multiple of 16."""

    def __init__(self, sizes, c_in, c_out, start=0, rest=0, seed=0, room=0, scale=0.01):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.sizes, self.start, groups = start + sum(sizes) + rest, list(sizes), start, len(sizes)
        pitch = (c_in + 15) // 16 * 16 + room
        ints = lambda *s: torch.randint(-128, 128, s, generator=gen, device="cuda", dtype=torch.int8)
        self.codes, self.kernel = ints(self.rows, pitch)[:, :c_in], ints(groups, c_out, pitch)[:, :, :c_in]
        self.scale = torch.exp(torch.randn(self.rows, generator=gen, device="cuda")) * scale
        self.scale[:start] = self.scale[start + sum(sizes):] = float("nan")
        self.kernel_scale = torch.exp(torch.randn((groups, c_out), generator=gen, device="cuda")) * scale
        self.kpos = kpos_of(sizes, start)

    def each(self):
        at = self.start
        for g, n in enumerate(self.sizes):
            yield g, slice(at, at + n)
            at += n

    def exact(self, fill=0.0):
        out = torch.full((self.rows, self.kernel.size(1)), fill, dtype=torch.float64, device="cuda")
        for g, rows in self.each():
            out[rows] = self.codes[rows].double() @ self.kernel[g].double().T * self.scale[rows].double()[:, None] * self.kernel_scale[g].double()
        return out


def allowed(exact, t):
    return exact.abs() * (torch.finfo(t).eps / 2 + 4 * 2.0 ** -24) + tiny(t)


SIZES = [  # sizes of the groups, c_in, c_out, rows before the first group, rows behind the last one
    ([1], 1, 1, 0, 0), ([1], 16, 8, 0, 0), ([1], 2048, 4096, 0, 0), ([3], 33, 7, 0, 0), ([1], 8192, 512, 0, 3),
    ([16], 128, 128, 0, 0), ([129], 257, 264, 0, 0), ([0, 5, 0], 100, 72, 2, 3), ([0, 0], 64, 64, 3, 0),
    ([40, 0, 1, 300, 7], 200, 136, 5, 9), ([700, 3, 512], 384, 1000, 0, 1), ([2500], 1000, 1496, 0, 0), ([5000, 3000], 512, 512, 0, 0),
    ([1] * 64, 512, 384, 0, 0), ([2, 1, 0, 3] * 30, 96, 48, 0, 0), ([30000], 64, 64, 0, 0), ([200], 20000, 130, 0, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_products(case, dtype):
    from fgms_b200 import backend
    sizes, c_in, c_out, start, rest = SIZES[case]
    t = TYPES[dtype]
    layer = Layer(sizes, c_in, c_out, start, rest, seed=case, scale=0.001)
    out = torch.full((layer.rows, c_out), 7.0, dtype=t, device="cuda")
    backend.fgms_grouped_i8_fwd_cuda(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, out, layer.kpos)
    exact = layer.exact(7.0)
    near(out, exact, allowed(exact, t))
    again = torch.full_like(out, 3.0)
    backend.fgms_grouped_i8_fwd_cuda(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, again, layer.kpos, zero_rest=True)
    inside = torch.zeros(layer.rows, dtype=torch.bool, device="cuda")
    inside[start:start + sum(sizes)] = True
    assert torch.equal(again[inside], out[inside]) and (again[~inside] == 0).all()
    assert backend.device_status() == 0


@pytest.mark.parametrize("c_in,c_out", [(100, 60), (1000, 333), (17, 128), (5, 5), (4, 16)])
@pytest.mark.parametrize("room", [1, 4, 7])
def test_rows_off_16_byte_boundaries_are_copied(c_in, c_out, room):
    from fgms_b200 import nn
    layer = Layer([50, 0, 33], c_in, c_out, seed=c_in, room=room, scale=0.001)
    exact = layer.exact()
    near(nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, layer.kpos, torch.float32), exact, allowed(exact, torch.float32))
    odd = torch.zeros(layer.codes.numel() + 3, dtype=torch.int8, device="cuda")[3:].view(layer.codes.shape)
    odd.copy_(layer.codes)
    near(nn.int8_linear(odd, layer.scale, layer.kernel.contiguous(), layer.kernel_scale, layer.kpos, torch.float32), exact, allowed(exact, torch.float32))


def test_sums_up_to_the_last_bit():
    """Sums that only an exact integer holds: 131071 products of the largest magnitude, which is 2^31 - 2^14, and their neighbours."""
    from fgms_b200 import nn
    k = 131071
    codes = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    kernel = torch.full((2, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    kernel[1, 5] = 127
    one = torch.ones(3, device="cuda")
    out = nn.int8_linear(codes, one, kernel, torch.ones(2, device="cuda"), dtype=torch.float32)
    want = codes[0].double() @ kernel.double().T
    assert want[0] == 2 ** 31 - 2 ** 14 and torch.equal(out, want.float().expand(3, 2))
    with pytest.raises(ValueError, match="131071"):
        nn.int8_linear(torch.zeros((1, k + 1), dtype=torch.int8, device="cuda"), one[:1], torch.zeros((1, k + 1), dtype=torch.int8, device="cuda"), one[:1])


def test_the_cut_changes_no_bit():
    """Rows computed alone (parts of a contraction shared by CTAs) and among many."""
    from fgms_b200 import nn
    layer = Layer([2000], 4096, 512, seed=3, scale=0.001)
    call = lambda r: nn.int8_linear(layer.codes[r], layer.scale[r], layer.kernel, layer.kernel_scale, dtype=torch.float32)
    whole = call(slice(None))
    for r in (slice(0, 1), slice(5, 9), slice(100, 140), slice(1000, 1300)):
        assert torch.equal(call(r), whole[r])


def test_scales_that_are_not_finite_stay_in_their_rows_and_channels():
    from fgms_b200 import nn
    layer = Layer([60], 64, 40, seed=4)
    want = nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale)
    layer.scale[7], layer.kernel_scale[0, 9] = float("nan"), float("inf")
    got = nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale)
    rows, channels = [i for i in range(60) if i != 7], [i for i in range(40) if i != 9]
    assert torch.isnan(got[7]).all() and not torch.isfinite(got[:, 9]).any()
    assert torch.equal(got[rows][:, channels], want[rows][:, channels])


def test_entries_of_kpos_out_of_order_and_out_of_range():
    from fgms_b200 import backend
    layer = Layer([10, 20, 30], 64, 64, seed=5)
    out = torch.zeros((60, 64), device="cuda")
    backend.device_status()
    bad = torch.tensor([0, 30, 10, 99], dtype=torch.int32, device="cuda")
    backend.fgms_grouped_i8_fwd_cuda(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, out, bad)
    assert backend.device_status() == 2
    layer.sizes = [30, 0, 30]
    near(out, layer.exact(), allowed(layer.exact(), torch.float32))


def test_on_a_stream_and_in_a_graph():
    from fgms_b200 import nn
    layer = Layer([200, 31, 0, 90], 130, 192, rest=9, seed=14, room=1)
    call = lambda: nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, layer.kpos)
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    graph.replay()
    assert torch.equal(got, want)
    layer.codes.neg_()
    layer.kpos.copy_(kpos_of([100, 100, 100, 10]))
    want = call()
    graph.replay()
    assert torch.equal(got, want)


def test_with_sms_kept_free():
    from fgms_b200 import _lib, nn
    layer = Layer([2000, 700], 512, 640, seed=6)
    call = lambda: nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, layer.kpos)
    want = call()
    _lib.lib.fgms_b200_set_reserved_sms(30)
    try:
        got = call()
    finally:
        _lib.lib.fgms_b200_set_reserved_sms(0)
    assert torch.equal(got, want)


def test_outputs_beyond_32_bits():
    from fgms_b200 import nn
    rows, c_out, tail = 560000, 4000, 100
    layer = Layer([rows], 48, c_out, seed=12, scale=0.001)
    for dtype in (torch.bfloat16, torch.float32):
        out = nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, layer.kpos, dtype)
        assert torch.equal(out[-tail:], nn.int8_linear(layer.codes[-tail:], layer.scale[-tail:].clone(), layer.kernel, layer.kernel_scale, dtype=dtype))
        del out


def test_a_block_for_serving():
    """Norm into 8 bits, a layer of groups in 8 bits, norm, a plain matrix: within the steps of the codes of the same in 64 bits.

    A code is off by half a scale at most, a value of a row by max / 254; an output by the sum over k of that times |w|, and the weights' the same way: what
    is allowed is that bound, evaluated in 64 bits, and the rounding of the output."""
    from fgms_b200 import nn
    gen = torch.Generator(device="cuda").manual_seed(8)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda")
    x, res, w = normal(90, 320).bfloat16(), normal(90, 320).bfloat16(), (1 + 0.1 * normal(320)).bfloat16()
    weight, kpos = (normal(3, 320, 200) * 320 ** -0.5).bfloat16(), kpos_of([50, 0, 40])
    layer = nn.Int8GroupedLinear(weight)
    codes, scale, h = nn.rms_norm_int8(x, w, residual=res)
    out = layer((codes, scale), kpos)
    assert out.dtype == torch.bfloat16
    total = x.double() + res.double()
    y = total / (total.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    for g, rows in ((0, slice(0, 50)), (2, slice(50, 90))):
        wg = weight[g].double()
        exact = y[rows] @ wg
        code_off = y[rows].abs().amax(1, keepdim=True) / 254 * 1.001 + 1e-5 * y[rows].abs()
        weight_off = wg.abs().amax(0) / 254 * 1.001
        bound = code_off @ wg.abs() + (y[rows].abs() + code_off).sum(1, keepdim=True) * weight_off
        near(out[rows], exact, bound * (1 + 2.0 ** -8) + exact.abs() * 2.0 ** -8 + 1e-30)
    assert torch.equal(layer(h, kpos), layer(nn.quantize_rows(h), kpos))
    assert set(layer.state_dict()) == {"kernel", "kernel_scale"}
    copy = nn.Int8GroupedLinear(torch.zeros_like(weight))
    copy.load_state_dict(layer.state_dict())
    assert torch.equal(copy((codes, scale), kpos), out)


def test_refusals():
    from fgms_b200 import backend, nn
    layer = Layer([10, 20], 64, 48)
    out = torch.zeros((30, 48), device="cuda", dtype=torch.bfloat16)
    call = backend.fgms_grouped_i8_fwd_cuda
    a = dict(codes=layer.codes, scale=layer.scale, kernel=layer.kernel, kernel_scale=layer.kernel_scale, out=out, kpos=layer.kpos)
    for change, text in [
        (dict(codes=layer.codes.float()), "int8"), (dict(kernel=layer.kernel.to(torch.uint8)), "int8"), (dict(codes=layer.codes[:, :32]), "channels"),
        (dict(codes=layer.codes.T.contiguous().T), "side by side"), (dict(scale=layer.scale[:9]), "30 float32"), (dict(scale=layer.scale.double()), "float32"),
        (dict(kernel_scale=layer.kernel_scale[0]), "float32"), (dict(kernel=layer.kernel[0]), "3 dimensions"), (dict(out=out[:, :40]), "contiguous"),
        (dict(out=out[:20]), "out must be"), (dict(out=out.double()), "unsupported"), (dict(kpos=None), "kpos is needed"), (dict(kpos=layer.kpos[:2]), "one entry more"),
        (dict(kpos=layer.kpos.long()), "int32"), (dict(codes=layer.codes.cpu()), "live on"), (dict(out=out.cpu()), "CUDA"),
        (dict(kernel=layer.kernel.transpose(1, 2).contiguous().transpose(1, 2)), "side by side"), (dict(kernel=layer.kernel[:1].expand(2, 48, 64)), "equally far"),
    ]:
        with pytest.raises(ValueError, match=text):
            call(**{**a, **change})
    with pytest.raises(TypeError, match="dtype"):
        nn.int8_linear(layer.codes, layer.scale, layer.kernel, layer.kernel_scale, layer.kpos, "bfloat16")
    with pytest.raises(ValueError, match="overlaps"):
        both = torch.zeros(30 * 64, dtype=torch.int8, device="cuda")
        out = both.view(torch.bfloat16).view(30, 32)
        call(both.view(30, 64), layer.scale, layer.kernel[:1, :32], layer.kernel_scale[:1, :32].contiguous(), out)
