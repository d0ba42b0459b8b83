"""Definitions in 64 bits of what stands between two layers, for the tests."""
import numpy as np
import torch


def philox(counter, key):
    """Philox 4x32-10 on arrays [n, 4] and [2] of 32-bit numbers (Salmon et al., SC 2011)."""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def kept(rows, width, p, seed, call, first=0):
    """What each value is multiplied by: 0, or the factor of those that are kept (a float64 array of the rows from `first` on)."""
    threshold = int(np.rint(p * 65536.0))
    if threshold == 65536:
        return np.zeros((rows, width))
    blocks = (width + 7) // 8
    counter = np.empty((rows, blocks, 4), dtype=np.uint64)
    counter[..., 0], counter[..., 1] = np.arange(blocks)[None, :], first + np.arange(rows)[:, None]
    counter[..., 2], counter[..., 3] = call & 0xFFFFFFFF, (call >> 32) & 0xFFFFFFFF
    words = philox(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    lots = np.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, blocks * 8)[:, :width]
    return (lots >= threshold) * (65536.0 / (65536 - threshold))


class Norm:
    """The norm and its gradients in 64 bits, and what a kernel may be off by.

    fp32 inside: a sum of n squares or products, in whatever order, is off by n 2^-24 of the sum of the magnitudes at most (the first order of
    n roundings); here a thread adds at most 32 values, a warp 5 times, a block 5 times more: 48.  16 more for the handful of operations beside
    it, the root and the quotient: SLACK.  What is stored is off by half a step of its type."""

    SLACK = 64 * 2.0 ** -24

    def __init__(self, x, weight, eps, residual=None, mask=None, exact_sum=False):
        d = lambda t: t.detach().double()
        self.unit = torch.finfo(x.dtype).eps / 2
        self.type = x.dtype
        dropped = d(x) if mask is None else torch.where(mask != 0, d(x) * mask, torch.zeros((), dtype=torch.float64, device=x.device))
        self.h = dropped if residual is None else dropped + d(residual)
        self.parts = dropped.abs() + (0 if residual is None else d(residual).abs())  # the fp32 sum h is off by a step of it
        self.mask, self.w = mask, d(weight)
        self.r = 1 / ((self.h ** 2).mean(1, keepdim=True) + eps).sqrt()
        self.y = self.h * self.r * self.w
        # of h where the backward reads it: stored rounded, or x itself
        exact = weight.dtype == torch.float32 and x.dtype != torch.float32  # computed once more
        self.stored = 0.0 if exact or (residual is None and mask is None) else self.unit

    def forward_allows(self):
        cancelled = 2.0 ** -23 * self.parts
        spread = (2 * self.h.abs() * cancelled).mean(1, keepdim=True) * self.r ** 2  # what r is off by, relative
        return self.y.abs() * (self.unit + self.SLACK + spread) + cancelled * self.r * self.w.abs() * (1 + self.unit) + tiny(self.type)

    def sum_allows(self):
        return self.h.abs() * self.unit + 2.0 ** -23 * self.parts + tiny(self.type)

    def backward(self, dy, dsum, weight_type):
        dy, dsum = dy.double(), (torch.zeros_like(self.h) if dsum is None else dsum.double())
        n, g = self.h * self.r, dy * self.w
        m, size = (g * n).mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
        dh = self.r * (g - n * m) + dsum
        off = self.stored + self.SLACK + 2.0 ** -23 * (self.parts * self.h.abs()).mean(1, keepdim=True) * self.r ** 2 * 2
        # h = a + b in fp32 is (a + b)(1 + d) where a = x factor is itself a(1 + d'): off by 2^-24 (|a + b| + |a|) <= 2^-23 parts, however small a + b is.
        # n = h r is then off by r 2^-23 parts beside what is relative to n, a product dy n by |dy| times that, and the mean m by the mean of |g| times that.
        # Where h is read as it was stored, a subnormal one is off by half a step of those.
        apart = (2.0 ** -23 * self.parts + (tiny(self.type) / 2 if self.stored else 0.0)) * self.r
        inside = self.r * (g.abs() * (self.SLACK + off) + n.abs() * (m.abs() + size) * 2 * off) + dsum.abs() * self.SLACK
        inside = inside + self.r * (apart * m.abs() + n.abs() * (g.abs() * apart).mean(1, keepdim=True))
        allows = dh.abs() * self.unit + inside * (1 + self.unit) + tiny(self.type)
        dx = dh if self.mask is None else torch.where(self.mask != 0, dh * self.mask, torch.zeros_like(dh))
        x_allows = allows if self.mask is None else allows * self.mask * (1 + 2.0 ** -23)
        dw, magnitude = (dy * n).sum(0), (dy * n).abs().sum(0)
        unit = torch.finfo(weight_type).eps / 2
        w_allows = dw.abs() * unit + (magnitude * (off.max() + dy.size(0) * 2.0 ** -24) + (dy.abs() * apart).sum(0)) * (1 + unit) + tiny(weight_type)
        return (dx, x_allows), (dh, allows), (dw, w_allows)


def tiny(t):
    """The step of a type's subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def near(got, exact, allowed):
    assert got.shape == exact.shape
    assert torch.isfinite(got).all()
    if got.numel():
        worst = ((got.double() - exact).abs() - allowed).max().item()
        assert worst <= 0, f"off by {worst} more than allowed"
