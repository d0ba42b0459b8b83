"""A training step of the encoder-decoder stack that ends with the update of its weights."""
import pytest
import torch

from fgms_b200 import unet, workloads

pytestmark = pytest.mark.gpu


def stack(**kw):
    wl = workloads.unet_workload(scenes=1, voxels=4000, grid=64)
    spec = unet.minkunet_spec(wl.c_in, wl.widths)
    weights = unet.unet_weights(spec, unet.build_unet_maps_host(wl.coords), wl.seed)
    maps = unet.build_unet_maps(torch.from_numpy(wl.coords).cuda())
    return unet.UNetStep(spec, maps, weights, torch.from_numpy(wl.feats).cuda(), torch.from_numpy(wl.grad_out).cuda(), **kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_run_ends_with_the_update(bits):
    """The first step from zero moments: master - lr (gradient / (|gradient| + eps) + decay master), every operation off by half a step; the
    layers' views show it, padded rows of the stem stay zero, and the next forward runs with it."""
    lr, decay, eps = 1e-3, 0.05, 1e-8
    step = stack(optimizer={"lr": lr, "weight_decay": decay, "eps": eps, "state_bits": bits})
    before = step._w_flat.clone()
    step.run()
    g, w = step.w_grad.double(), before.double()
    want = w * (1 - lr * decay) - lr * g / (g.abs() + eps)
    state = step.optimizer.state[step._w_flat]
    assert state["step"].tolist() == [1, 0] and state["master"].dtype == torch.float32
    assert ((state["master"].double() - want).abs() <= want.abs() * 2.0 ** -22 + lr * 2.0 ** -19).all()
    assert torch.equal(step._w_flat, state["master"].half())
    assert step.weights[3].data_ptr() >= step._w_flat.data_ptr() and not torch.equal(step._w_flat, before)
    assert not step._w_run[0][:, step._cin0:].any()
    out = step.val[step.out_name].clone()
    step.run()
    assert not torch.equal(out, step.val[step.out_name]) and state["step"].tolist() == [2, 0]


def test_without_an_optimizer_nothing_changes():
    step = stack()
    before = step._w_flat.clone()
    step.run()
    assert torch.equal(step._w_flat, before) and step.optimizer is None
    with pytest.raises(ValueError, match="optimizer"):
        step.update()


def test_the_step_with_its_update_in_a_graph():
    """Replays go on where the steps before them ended.  The gradients of the stack are added up by atomics, so two runs differ in their last
    bits; the count of the steps and a weight whose gradient is zero do not."""
    step = stack(optimizer={"lr": 1e-2, "weight_decay": 0.5})
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    graph.replay()
    state = step.optimizer.state[step._w_flat]
    assert torch.isfinite(step._w_flat).all() and torch.equal(step._w_flat, state["master"].half())
    # Steps of 0.01 on weights of about 0.1 make 25 layers without a normalisation grow: the largest activation of the last one is 23, 4400 behind one step,
    # and beyond fp16 behind two, with or without a graph.  So the steps after that are only counted.
    for _ in range(2):
        graph.replay()
    assert state["step"].tolist() == [4, 0]


def test_module_with_the_optimizer():
    """``nn.SparseUNet`` and ``optim.AdamW`` as a training loop uses them: one launch for the 25 layers."""
    from fgms_b200 import backend, nn, optim
    wl = workloads.unet_workload(scenes=1, voxels=3000, grid=64)
    spec = unet.minkunet_spec(wl.c_in, wl.widths)
    maps = unet.build_unet_maps(torch.from_numpy(wl.coords).cuda())
    net = nn.SparseUNet(spec)
    net.load_weights(unet.unet_weights(spec, unet.build_unet_maps_host(wl.coords), wl.seed))
    opt = optim.AdamW(net.parameters(), lr=1e-3, state_bits=8)
    feats, grad = torch.from_numpy(wl.feats).cuda(), torch.from_numpy(wl.grad_out).cuda()
    before = [p.detach().clone() for p in net.parameters()]
    net(feats, maps).backward(grad)
    launches = backend.launch_count()
    opt.step()
    assert backend.launch_count() - launches == 1
    for p, b in zip(net.parameters(), before):
        want = b.double() * (1 - 1e-5) - 1e-3 * p.grad.double() / (p.grad.double().abs() + 1e-8)
        assert ((p.double() - want).abs() <= want.abs() * 2.0 ** -11 + 1e-3 * 2.0 ** -19 + 2.0 ** -25).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_take_the_steps_of_the_formula(bits):
    """Each replay's step in 64 bits from the master and the moments before it and from the gradient that the replay itself left, which holds although the
    gradients' last bits differ from run to run.  Differences: a moment is off by 2^-22 of its terms, the update by 2^-20 of its size with the
    terms of m in m's place, the value by 2^-22 of itself."""
    lr, b1, b2, eps, decay = 1e-4, 0.9, 0.999, 1e-8, 0.1
    step = stack(optimizer={"lr": lr, "betas": (b1, b2), "eps": eps, "weight_decay": decay, "state_bits": bits})
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    state = step.optimizer.state[step._w_flat]

    def moment(name):
        held = state[name].float().double().view(-1)
        if bits == 32:
            return held
        return held * state[name + "_scale"].double().repeat_interleave(128)[:held.numel()]
    for t in (2, 3, 4):
        w, m, v = state["master"].double().view(-1), moment("exp_avg"), moment("exp_avg_sq")
        feats_in = step.val[step.out_name].clone()
        step.w_grad.zero_()
        graph.replay()
        g = step.w_grad.double().view(-1)
        assert g.any() and not torch.equal(feats_in, step.val[step.out_name])  # this replay's own forward and gradient
        terms = b1 * m.abs() + (1 - b1) * g.abs()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        rate, denominator = lr / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt() + eps
        want = w * (1 - lr * decay) - rate * m / denominator
        now = state["master"].double().view(-1)
        assert ((now - want).abs() <= w.abs() * 2.0 ** -22 + rate * terms / denominator * 2.0 ** -20 + 2.0 ** -149).all()
        moved = (now - w).abs()
        assert (moved[g != 0] > 0).double().mean() > 0.99 and torch.equal(step._w_flat, state["master"].half())
        assert state["step"].tolist() == [t, 0]


@pytest.mark.parametrize("set_to_none", [True, False])
def test_the_update_is_taken_behind_zero_grad(set_to_none):
    """The optimizer is a PyTorch one, and loops over those clear gradients: the step's own, which every backward overwrites, are used all the same."""
    step = stack(optimizer={"lr": 1e-4})
    for t in (1, 2):
        before = step._w_flat.clone()
        step.optimizer.zero_grad(set_to_none=set_to_none)
        step.run()
        assert step.w_grad.any() and not torch.equal(step._w_flat, before)
        assert step.optimizer.state[step._w_flat]["step"].tolist() == [t, 0]
