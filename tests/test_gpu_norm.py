"""Norm with the residual's addition, dropout and rows in 8 bits against their definitions in 64 bits (``layers_ref``, which also derives what is allowed)."""
import math

import pytest
import torch

from tests.layers_ref import Norm, kept, near, tiny

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SEED = 0x5EED_0123_4567
# rows and widths: one value; less than a chunk; a warp's rows and their borders; a block's, odd and even, one chunk a thread and more; the widest
SHAPES = [(1, 1), (3, 5), (9, 8), (130, 64), (17, 255), (5, 256), (33, 257), (700, 512), (2, 513), (301, 1000), (64, 1001), (1, 2048), (400, 2056),
          (1, 8192), (160, 8200), (3, 16384), (150, 16390), (2, 32768)]


def made(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


class Case:
    def __init__(self, dtype, rows, width, weight="same", seed=0):
        t = TYPES[dtype]
        self.x, self.res = made(seed, rows, width, dtype=t), (made(seed + 1, rows, width) * torch.exp(made(seed + 2, rows, 1))).to(t)
        self.w = (1 + 0.3 * made(seed + 3, width)).to(t if weight == "same" else torch.float32)
        self.dy, self.dsum = made(seed + 4, rows, width, dtype=t), made(seed + 5, rows, width, dtype=t)


def mask_of(case, p, call=0, seed=SEED):
    return torch.from_numpy(kept(*case.x.shape, p, seed, call)).cuda()


@pytest.mark.parametrize("dtype,weight", [("fp32", "same"), ("fp16", "same"), ("bf16", "fp32"), ("bf16", "same"), ("fp16", "fp32")])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward_and_gradients(dtype, weight, rows, width):
    from fgms_b200 import nn
    c = Case(dtype, rows, width, weight, seed=rows + width)
    for residual, p in ((None, 0.0), (c.res, 0.0), (c.res, 0.25), (None, 0.25)):
        rng = nn.rng_state(SEED)
        x, w = c.x.clone().requires_grad_(), c.w.clone().requires_grad_()
        res = None if residual is None else residual.clone().requires_grad_()
        got = nn.rms_norm(x, w, 1e-5, residual=res, dropout=p, rng=rng if p else None)
        ref = Norm(c.x, c.w, 1e-5, residual, mask_of(c, p) if p else None)
        out = got if residual is None else got[0]
        near(out.detach(), ref.y, ref.forward_allows())
        if residual is None:
            grads, dsum = torch.autograd.grad(out, (x, w), c.dy), None
        else:
            near(got[1].detach(), ref.h, ref.sum_allows())
            dsum = c.dsum
            grads = torch.autograd.grad(got, (x, w, res), (c.dy, dsum))
        dx, dres, dw = ref.backward(c.dy, dsum, c.w.dtype)
        near(grads[0], *dx)
        near(grads[1], *dw)
        if residual is not None:
            near(grads[2], *dres)
        assert rng.tolist() == [SEED, 1 if p else 0, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_an_output_in_8_bits(dtype, rows, width):
    from fgms_b200 import nn
    c = Case(dtype, rows, width, seed=3 * rows + width)
    ref = Norm(c.x, c.w, 1e-5, c.res)
    codes, scale, total = nn.rms_norm_int8(c.x, c.w, 1e-5, residual=c.res)
    near(total, ref.h, ref.sum_allows())
    assert codes.dtype == torch.int8 and codes.stride(0) % 16 == 0 or rows == 1
    allowed = ref.forward_allows() + ref.y.abs() * 2.0 ** -22 - ref.y.abs() * ref.unit  # y in fp32: no rounding to the rows' type
    largest = ref.y.abs().amax(1)
    near(scale, largest / 127, (allowed.amax(1) + largest * 2.0 ** -22) / 127)
    near(codes.double() * scale.double()[:, None], ref.y, scale.double()[:, None] * (0.5 + 2.0 ** -16) + allowed)
    assert (codes.int().abs().amax(1) == 127).all()
    codes, scale = nn.quantize_rows(c.x)
    x = c.x.double()
    near(scale, x.abs().amax(1) / 127, x.abs().amax(1) * 2.0 ** -23 / 127 * 2)
    near(codes.double() * scale.double()[:, None], x, scale.double()[:, None] * (0.5 + 2.0 ** -16))


def test_rows_in_8_bits_that_are_zero_tiny_or_not_finite():
    from fgms_b200 import nn
    x = made(1, 6, 300)
    x[1] = 0.0
    x[2] *= 1e-35
    x[3, 7] = float("nan")
    x[4, 299] = float("-inf")
    codes, scale = nn.quantize_rows(x)
    assert (codes[1:5] == 0).all() and (scale[1:3] == 0).all() and torch.isnan(scale[3:5]).all()
    assert (codes[0].int().abs().max() == 127) and (codes[5].int().abs().max() == 127)
    codes, scale = nn.rms_norm_int8(x, torch.ones(300, device="cuda"))
    assert torch.isnan(scale[3:5]).all() and scale[1] == 0 and (codes[[1, 3, 4]] == 0).all()
    assert (codes[2].int().abs().max() <= 127) and scale[2] >= 0
    w = torch.ones(300, device="cuda")
    w[5] = float("inf")
    assert torch.isnan(nn.rms_norm_int8(x, w)[1][[0, 5]]).all()


def test_values_of_rows_that_are_not_finite_stay_in_their_rows():
    from fgms_b200 import nn
    c = Case("bf16", 40, 700)
    want = nn.rms_norm(c.x, c.w, residual=c.res)
    c.x[7, 3], c.x[8, 699], c.x[30] = float("nan"), float("inf"), float("-inf")
    got = nn.rms_norm(c.x, c.w, residual=c.res)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 8, 30]] = True
    assert all(torch.equal(a[~bad], b[~bad]) for a, b in zip(got, want))
    assert torch.isnan(got[0][7]).all() and torch.isnan(got[0][30]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,p", [(1, 1, 0.5), (7, 3, 0.3), (100, 260, 0.5), (1000, 1001, 0.1), (5000, 64, 0.9), (3, 100000, 0.05), (2049, 4096, 0.25), (64, 64, 1.0),
                                          (64, 64, 0.0), (64, 64, 1e-6)])
def test_dropout(dtype, rows, width, p):
    from fgms_b200 import nn
    c = Case(dtype, rows, width, seed=rows)
    unit = torch.finfo(TYPES[dtype]).eps / 2
    rng = nn.rng_state(SEED)
    for call, residual in enumerate((None, c.res, c.res)):
        x = c.x.clone().requires_grad_()
        res = None if residual is None else residual.clone().requires_grad_()
        out = nn.dropout(x, p, rng, residual=res)
        m = mask_of(c, p, call)
        ref = c.x.double() * m + (0 if residual is None else residual.double())
        size = (c.x.double() * m).abs() + (0 if residual is None else residual.double().abs())
        near(out.detach(), ref, ref.abs() * unit + size * 2.0 ** -23 + tiny(TYPES[dtype]))
        if residual is None:
            assert torch.equal(out.detach() == 0, (m == 0) | (c.x == 0))
            grads = torch.autograd.grad(out, (x,), c.dy)
        else:
            grads = torch.autograd.grad(out, (x, res), c.dy)
            assert torch.equal(grads[1], c.dy)
        near(grads[0], c.dy.double() * m, (c.dy.double() * m).abs() * (unit + 2.0 ** -23) + tiny(TYPES[dtype]))
    assert rng.tolist() == [SEED, 3, 0]


def test_dropped_values_are_gone_whatever_they_were():
    from fgms_b200 import nn
    c = Case("fp32", 50, 90)
    m = mask_of(c, 0.5) == 0
    c.x[m] = float("nan")
    out = nn.dropout(c.x, 0.5, nn.rng_state(SEED))
    assert (out[m] == 0).all() and torch.isfinite(out).all()
    y, h = nn.rms_norm(c.x, c.w, residual=c.res, dropout=0.5, rng=nn.rng_state(SEED))
    assert torch.isfinite(y).all() and torch.equal(h[m], c.res[m])


def test_the_call_number_goes_beyond_32_bits():
    from fgms_b200 import nn
    c = Case("fp32", 20, 40)
    call = 2 ** 32 + 9
    rng = torch.tensor([SEED, call, 0], device="cuda")
    assert torch.equal(nn.dropout(c.x, 0.5, rng) != 0, mask_of(c, 0.5, call) != 0) and rng.tolist() == [SEED, call + 1, 0]


def test_gradients_against_differences():
    """Central differences of the definition in 64 bits agree with the formulas that the kernels are held to."""
    from tests.layers_ref import Norm as N
    c = Case("fp32", 4, 24)
    mask = mask_of(c, 0.5)
    f = lambda x, w, res: ((N(x, w, 1e-5, res, mask).y * c.dy.double()).sum() + (N(x, w, 1e-5, res, mask).h * c.dsum.double()).sum()).item()
    (dx, _), (dres, _), (dw, _) = N(c.x, c.w, 1e-5, c.res, mask).backward(c.dy, c.dsum, torch.float32)
    x, w, res = c.x.double(), c.w.double(), c.res.double()
    for t, grad in ((x, dx), (res, dres), (w, dw)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 5):
            keep, step = flat[i].item(), 1e-5
            flat[i] = keep + step
            up = f(x, w, res)
            flat[i] = keep - step
            down = f(x, w, res)
            flat[i] = keep
            assert abs((up - down) / (2 * step) - grad.view(-1)[i].item()) <= 1e-6 * (1 + abs(grad.view(-1)[i].item()))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_alignment_and_shapes(dtype):
    from fgms_b200 import backend, nn
    t = TYPES[dtype]
    c = Case(dtype, 70, 264)
    want, total = nn.rms_norm(c.x, c.w, residual=c.res)
    wide = made(9, 70, 900, dtype=t)
    for at in (0, 1, 2, 3, 5, 7, 8, 271):  # on and off 16-byte boundaries
        x, out = wide[:, at:at + 264], wide[:, at + 300:at + 564]
        x.copy_(c.x)
        keep = wide.clone()
        backend.fgms_rms_norm_cuda(x, c.w, out, residual=c.res)
        assert torch.equal(out, want)
        keep[:, at + 300:at + 564] = want
        assert torch.equal(wide, keep)  # nothing beside the columns
    inplace, res = c.x.clone(), c.res.clone()
    backend.fgms_rms_norm_cuda(inplace, c.w, inplace, residual=res, residual_out=res)
    assert torch.equal(inplace, want) and torch.equal(res, total)
    for shape in ((264,), (2, 5, 7, 264)):
        x, r = c.x.view(-1)[:math.prod(shape)].view(shape), c.res.view(-1)[:math.prod(shape)].view(shape)
        y, h = nn.rms_norm(x, c.w, residual=r)
        assert y.shape == h.shape == shape and torch.equal(y.view(-1, 264), want[:y.numel() // 264])
    assert torch.equal(nn.rms_norm(c.x.T.contiguous().T, c.w, residual=c.res)[0], want)
    codes, scale = nn.quantize_rows(wide[:, 3:103])
    again = torch.full((70, 100), 9, dtype=torch.int8, device="cuda")
    scales = torch.empty(70, device="cuda")
    backend.fgms_quantize_rows_cuda(wide[:, 3:103], again, scales)
    assert torch.equal(codes, again) and torch.equal(scale, scales)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 7, 9, 31, 255, 257, 1003, 2046, 5001, 9999, 20001])
def test_rows_off_every_boundary(dtype, width):
    """Rows at every distance from a 16-byte boundary, on both sides of what stays as it was: the same bits as aligned rows, nothing else written."""
    from fgms_b200 import backend, nn
    c = Case(dtype, 21, width, seed=width)
    rng, rstd, used = nn.rng_state(SEED), torch.empty(21, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
    room = (width + 39) // 8 * 8
    plain = lambda t: torch.zeros((21, room), dtype=t.dtype, device="cuda")[:, :width].copy_(t)  # rows on boundaries
    x, res, dy = plain(c.x), plain(c.res), plain(c.dy)
    out, total, dx, dropped = plain(c.x), plain(c.x), plain(c.x), plain(c.x)
    dw = torch.empty_like(c.w)

    def run(x, res, dy, out, total, dx, dropped):
        backend.fgms_rms_norm_cuda(x, c.w, out, residual=res, residual_out=total, rstd=rstd, dropout=0.25, rng=rng, rng_used=used)
        backend.fgms_rms_norm_bwd_cuda(dy, total, c.w, rstd, x_grad=dx, weight_grad=dw, h_grad=res, dropout=0.25, rng_used=used)
        backend.fgms_dropout_cuda(x, dropped, 0.25, rng, residual=dy)
        return dw.clone()

    want = run(x, res, dy, out, total, dx, dropped)
    for shift in (1, 2, 3, 4, 5, 6, 7):
        rng.copy_(nn.rng_state(SEED))
        flat = [torch.full((21 * (width + 3) + 16,), 5.0, dtype=c.x.dtype, device="cuda") for _ in range(7)]
        views = [f[shift:shift + 21 * (width + 3)].view(21, width + 3)[:, :width] for f in flat]  # every row at another distance
        for v, t in zip(views, (x, res, dy)):
            v.copy_(t)
        assert torch.equal(run(*views), want)
        assert all(torch.equal(a, b) for a, b in zip(views, (x, res, dy, out, total, dx, dropped)))
        for f, v in zip(flat, views):
            v.fill_(5.0)
            assert (f == 5.0).all()


def test_gradients_in_pieces():
    """What is asked for alone is what it is together; gradients that are expanded; a sum whose gradient alone is given."""
    from fgms_b200 import backend, nn
    c = Case("bf16", 90, 600, "fp32")
    rng = nn.rng_state(SEED)
    leaves = [t.clone().requires_grad_() for t in (c.x, c.w, c.res)]
    y, h = nn.rms_norm(leaves[0], leaves[1], residual=leaves[2], dropout=0.5, rng=rng)
    both = torch.autograd.grad((y, h), leaves, (c.dy, c.dsum), retain_graph=True)
    for i in range(3):
        (one,) = torch.autograd.grad((y, h), (leaves[i],), (c.dy, c.dsum), retain_graph=True)
        assert torch.equal(one, both[i])
    (only,) = torch.autograd.grad(h, (leaves[2],), c.dsum, retain_graph=True)
    assert torch.equal(only, c.dsum)
    ones = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(ones, torch.autograd.grad(y, leaves, torch.ones_like(y))))
    rstd, used = torch.empty(90, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
    out, total = torch.empty_like(c.x), torch.empty_like(c.x)
    backend.fgms_rms_norm_cuda(c.x, c.w, out, residual=c.res, residual_out=total, rstd=rstd, dropout=0.5, rng=nn.rng_state(SEED), rng_used=used)
    assert torch.equal(out, y) and torch.equal(total, h) and used.tolist() == [SEED, 0]
    dx, dres, dw = c.dy.clone(), torch.empty_like(c.x), torch.empty_like(c.w)
    backend.fgms_rms_norm_bwd_cuda(dx, None, c.w, rstd, x_grad=dx, weight_grad=dw, h_grad=c.dsum, residual_grad=dres, dropout=0.5, rng_used=used, x=c.x,
                                   residual=c.res)  # dx over dy
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1]) and torch.equal(dres, both[2])
    ref = Norm(c.x, c.w, 1e-6, c.res, mask_of(c, 0.5))
    ref.stored = ref.unit  # from the sum as it was stored
    grads = torch.empty_like(c.x), torch.empty_like(c.x), torch.empty_like(c.w)
    backend.fgms_rms_norm_bwd_cuda(c.dy, total, c.w, rstd, x_grad=grads[0], residual_grad=grads[1], weight_grad=grads[2], h_grad=c.dsum, dropout=0.5, rng_used=used)
    for got, want in zip(grads, ref.backward(c.dy, c.dsum, torch.float32)):
        near(got, *want)
    for args in (dict(h=None), dict(h=total, x=c.x), dict(h=total, residual=c.res)):
        with pytest.raises(ValueError, match="either h or x|goes with x"):
            backend.fgms_rms_norm_bwd_cuda(c.dy, weight=c.w, rstd=rstd, x_grad=grads[0], **args)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        y, h = nn.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        grads = torch.autograd.grad((y * y).sum(), leaves, create_graph=True)
        sum(g.float().sum() for g in grads).backward()
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        (g,) = torch.autograd.grad((nn.dropout(leaves[0], 0.5, rng) ** 2).sum(), leaves[:1], create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("weight", ["same", "fp32"])
@pytest.mark.parametrize("residual", [False, True])
def test_a_weight_that_is_frozen(weight, residual):
    from fgms_b200 import nn
    c = Case("bf16", 50, 130, weight, seed=3)
    x, res = c.x.clone().requires_grad_(), c.res.clone().requires_grad_() if residual else None
    got = nn.rms_norm(x, c.w, 1e-5, residual=res, dropout=0.5, rng=nn.rng_state(SEED))
    ref = Norm(c.x, c.w, 1e-5, c.res if residual else None, mask_of(c, 0.5))
    ref.stored = ref.unit
    leaves = (x, res) if residual else (x,)
    grads = torch.autograd.grad(got[0] if residual else got, leaves, c.dy)
    for g, want in zip(grads, ref.backward(c.dy, None, torch.float32)):
        near(g, *want)


def test_no_rows():
    from fgms_b200 import nn
    x, w, rng = torch.zeros((0, 64), device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True), nn.rng_state(1)
    y, h = nn.rms_norm(x, w, residual=torch.zeros_like(x), dropout=0.5, rng=rng)
    gx, gw = torch.autograd.grad((y.sum() + h.sum()), (x, w))
    assert gx.shape == (0, 64) and (gw == 0).all() and rng.tolist() == [1, 0, 0]
    assert nn.dropout(x, 0.5, rng).shape == (0, 64) and rng.tolist() == [1, 0, 0]
    codes, scale = nn.quantize_rows(x.detach())
    assert codes.shape == (0, 64) and scale.shape == (0,)


def test_the_same_bits_on_every_run_and_with_sms_kept_free():
    from fgms_b200 import _lib, nn
    c = Case("fp16", 3000, 1024, "fp32")

    def step():
        leaves = [t.clone().requires_grad_() for t in (c.x, c.w, c.res)]
        y, h = nn.rms_norm(leaves[0], leaves[1], residual=leaves[2], dropout=0.1, rng=nn.rng_state(SEED))
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (c.dy, c.dsum)))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    _lib.lib.fgms_b200_set_reserved_sms(20)
    try:
        got = step()
    finally:
        _lib.lib.fgms_b200_set_reserved_sms(0)
    ref = Norm(c.x, c.w, 1e-6, c.res, mask_of(c, 0.1))
    for i in (0, 1, 2, 4):
        assert torch.equal(got[i], want[i])
    near(got[3], *ref.backward(c.dy, c.dsum, torch.float32)[2])  # other shares of the rows


def test_replays_drop_other_values_and_streams_do_not_disturb():
    from fgms_b200 import nn
    c = Case("bf16", 300, 520)
    leaves = [t.clone().requires_grad_() for t in (c.x, c.w, c.res)]
    rng = nn.rng_state(SEED)

    def step(rng):
        y, h = nn.rms_norm(leaves[0], leaves[1], residual=leaves[2], dropout=0.3, rng=rng)
        z = nn.dropout(y, 0.5, rng, residual=h)
        return (z.detach(), *torch.autograd.grad(z, leaves, c.dy))

    want = [step(rng) for _ in range(4)]  # calls 0..7
    rng.copy_(nn.rng_state(SEED))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(rng)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(rng)
    assert rng.tolist() == [SEED, 2, 0]  # captured, not run
    for i in (1, 2, 3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
    assert rng.tolist() == [SEED, 8, 0]


def test_values_beyond_32_bits():
    """2.2e9 values: the last rows are what they are by themselves, and so are their gradients and what is dropped of them."""
    from fgms_b200 import backend, nn
    rows, width, tail = 67000, 32760, 8
    x = torch.empty((rows, width), dtype=torch.float16, device="cuda")
    x.fill_(0.5)
    x[-tail:] = made(1, tail, width, dtype=torch.float16)
    w = (1 + 0.3 * made(2, width)).half()
    y = nn.rms_norm(x, w)
    assert torch.equal(y[-tail:], nn.rms_norm(x[-tail:].clone(), w))
    out, rng, used = y, nn.rng_state(SEED), torch.empty(2, dtype=torch.int64, device="cuda")
    backend.fgms_dropout_cuda(x, out, 0.25, rng, rng_used=used)
    m = torch.from_numpy(kept(tail, width, 0.25, SEED, 0, first=rows - tail)).cuda()
    want = x[-tail:].double() * m
    near(out[-tail:], want, want.abs() * (2.0 ** -11 + 2.0 ** -23) + tiny(torch.float16))
    backend.fgms_dropout_bwd_cuda(out, out, 0.25, used)  # twice the same lots: dropped where it was dropped
    assert torch.equal(out[-tail:] == 0, (m == 0) | (x[-tail:] == 0))
    rstd = torch.ones(rows, device="cuda")
    dx = torch.empty((tail, width), dtype=torch.float16, device="cuda")
    backend.fgms_rms_norm_bwd_cuda(out[-tail:].clone(), x[-tail:].clone(), w, rstd[-tail:].clone(), x_grad=dx)
    backend.fgms_rms_norm_bwd_cuda(out, x, w, rstd, x_grad=out)  # over what flows in
    assert torch.equal(out[-tail:], dx)
    codes, scale = nn.quantize_rows(x)
    few = nn.quantize_rows(x[-tail:].clone())
    assert torch.equal(codes[-tail:], few[0]) and torch.equal(scale[-tail:], few[1])


def test_modules():
    from fgms_b200 import nn
    c = Case("bf16", 40, 128)
    norm, drop = nn.RMSNorm(128, dropout=0.5, seed=SEED), nn.Dropout(0.5, seed=SEED)
    mask = mask_of(c, 0.5)
    ref = Norm(c.x, norm.weight, 1e-6, c.res, mask)
    y, h = norm(c.x, c.res)
    near(y.detach(), ref.y, ref.forward_allows())
    near(h.detach(), ref.h, ref.sum_allows())
    y.float().sum().backward()
    assert norm.weight.grad.shape == (128,)
    assert torch.equal(drop(c.x) != 0, (mask != 0) & (c.x != 0))
    norm.eval(), drop.eval()
    assert torch.equal(norm(c.x), nn.rms_norm(c.x, norm.weight)) and drop(c.x) is c.x and torch.equal(drop(c.x, c.res), c.res + c.x)
    assert set(norm.state_dict()) == {"weight", "rng"} and norm.rng.tolist() == [SEED, 1, 0]


def test_refusals():
    from fgms_b200 import backend, nn
    c = Case("bf16", 10, 64)
    rng = nn.rng_state(1)
    for call, text in [
        (lambda: nn.rms_norm(c.x, c.w.half()), "weight must have dtype"), (lambda: nn.rms_norm(c.x, c.w[:60]), "weight must have 64"),
        (lambda: nn.rms_norm(c.x, c.w, residual=c.res[:5]), "shape of x"), (lambda: nn.rms_norm(c.x, c.w, residual=c.res.float()), "dtype"),
        (lambda: nn.rms_norm(c.x, c.w.cpu()), "must live on"), (lambda: nn.rms_norm(c.x, c.w, dropout=0.5), "rng is needed"),
        (lambda: nn.rms_norm(c.x, c.w, dropout=1.5, rng=rng), "probability"), (lambda: nn.rms_norm(c.x, c.w, eps=-1.0), "eps"),
        (lambda: nn.rms_norm(c.x.double(), c.w), "unsupported feature dtype"), (lambda: nn.rms_norm(c.x.int(), c.w), "unsupported feature dtype"),
        (lambda: nn.dropout(c.x, 0.5, rng.int()), "dtype"), (lambda: nn.dropout(c.x, 0.5, rng[:2]), "3 values"), (lambda: nn.dropout(c.x, 0.5, rng.cpu()), "live on"),
        (lambda: nn.dropout(c.x, -0.1, rng), "probability"), (lambda: nn.dropout(c.x, 0.5, rng, residual=c.res[:, :8]), "shape of x"),
        (lambda: nn.rms_norm_int8(c.x.clone().requires_grad_(), c.w), "no_grad"), (lambda: nn.quantize_rows(c.x[0]), "2 dimensions"),
        (lambda: nn.rms_norm(torch.zeros((2, 32776), device="cuda"), torch.ones(32776, device="cuda")), "width 32776"),
        (lambda: backend.fgms_rms_norm_cuda(c.x, c.w, c.x.T.contiguous().T), "side by side"),
        (lambda: backend.fgms_rms_norm_cuda(c.x, c.w, c.x[:1].expand(10, 64)), "overlap"),
        (lambda: backend.fgms_rms_norm_cuda(c.x, c.w, c.x.clone(), scale=torch.zeros(10, device="cuda")), "out must have dtype"),
        (lambda: backend.fgms_rms_norm_cuda(c.x, c.w, c.res, residual_out=c.res), "two outputs"),
        (lambda: backend.fgms_rms_norm_bwd_cuda(c.dy, c.x, c.w, torch.zeros(9, device="cuda")), "10 values"),
        (lambda: backend.fgms_dropout_bwd_cuda(c.dy, c.x, 0.5, rng), "2 values"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    assert rng.tolist() == [1, 0, 0]


def test_autograd_notices_what_was_written():
    from fgms_b200 import backend, nn
    c = Case("fp32", 20, 30)
    x = c.x.clone().requires_grad_()
    y = nn.rms_norm(x, c.w)
    with torch.no_grad():
        backend.fgms_dropout_cuda(c.res, x, 0.5, nn.rng_state(1))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
