"""Modules that drop values have seeds of their own (no GPU: their states alone)."""
import pytest
import torch

from fgms_b200 import nn


def seeds(**kw):
    return [m.rng[0].item() for m in (nn.Dropout(0.5, device="cpu", **kw), nn.Dropout(0.5, device="cpu", **kw), nn.RMSNorm(8, dropout=0.5, device="cpu", **kw),
                                      nn.RMSNorm(8, dropout=0.5, device="cpu", **kw))]


def test_modules_at_their_defaults_have_different_seeds():
    torch.manual_seed(1)
    first = seeds()
    assert len(set(first)) == 4 and all(0 <= s < 2 ** 63 for s in first)
    assert not set(first) & set(seeds())
    torch.manual_seed(1)
    assert seeds() == first
    torch.manual_seed(2)
    assert not set(first) & set(seeds())


def test_a_seed_that_is_given_is_the_seed():
    torch.manual_seed(3)
    want = torch.rand(4)
    torch.manual_seed(3)
    assert seeds(seed=0) == [0] * 4 and seeds(seed=2 ** 63 - 1) == [2 ** 63 - 1] * 4
    nn.RMSNorm(8, device="cpu")  # drops nothing: no seed is drawn
    assert torch.equal(torch.rand(4), want)
    for bad in (-1, 2 ** 63):
        with pytest.raises(ValueError, match="seed"):
            nn.Dropout(0.5, device="cpu", seed=bad)


def test_every_rank_has_its_own(monkeypatch):
    monkeypatch.setattr(torch.distributed, "is_initialized", lambda: True)
    found = []
    for rank in range(16):
        monkeypatch.setattr(torch.distributed, "get_rank", lambda: rank)
        torch.manual_seed(4)
        found += seeds()
        torch.manual_seed(4)
        assert seeds(seed=5) == [5] * 4
    assert len(set(found)) == 64 and all(0 <= s < 2 ** 63 for s in found)


def test_states_of_a_segment_that_is_computed_again():
    a, b = nn.rng_state(1, "cpu"), nn.Dropout(0.5, device="cpu", seed=2)
    layers = torch.nn.Sequential(b, nn.RMSNorm(8, device="cpu"))  # of which one has no state
    forward, again = nn.recomputed(a, layers, b.rng)
    a[1], b.rng[1] = 4, 5
    with forward:
        a[1] += 2
        b.rng[1] += 1
    a[1] += 10
    for _ in range(2):
        with pytest.raises(RuntimeError, match="stopped"):
            with again:
                assert a.tolist() == [1, 4, 0] and b.rng.tolist() == [2, 5, 0]
                a[1] += 1
                raise RuntimeError("stopped")
        assert a.tolist() == [1, 16, 0] and b.rng.tolist() == [2, 6, 0]
    for bad in (3, None, torch.zeros(3), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="states of rng_state"):
            nn.recomputed(bad)
