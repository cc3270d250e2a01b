"""Mirror of the reference's `nn` helpers that the configs and known-answer tests use:
Linear / LinearWithWeights (src/nn/linear.rs:5-49), Sequential (src/nn/sequential.rs),
Sigmoid / ReLU / Softmax (src/nn/activations), RMS / LayerNorm (src/nn/norm) and SGD
(src/nn/optimizers/sgd.rs:3-28), plus the two helpers upstream lists as missing (mse_loss, Tensor.abs) and the layers
over the device's transformer operators (ResidualRMS, Rotary, SelfAttention).  Each `f` composes Tensor ops exactly as upstream does,
so the IR reaching the device has the same shape.
"""
from __future__ import annotations

import numpy as np

from . import autodiff
from .autodiff import Tensor, f32


class Module:
    def params(self) -> list:
        return []

    def f(self, x: Tensor) -> Tensor:
        raise NotImplementedError


class Linear(Module):
    """`res = dot(x, w); res += b` (src/nn/linear.rs:20-28).  `Linear(inp, out, bias)` draws
    standard-normal weights like upstream; pass `rng` for a seeded draw."""

    def __init__(self, inp=None, out=None, bias=True, *, w: Tensor = None, b: Tensor = None, rng=None):
        if w is None:
            w = autodiff.randn([inp, out], rng)
            b = autodiff.randn([out], rng) if bias else None
        self.w, self.b = w, b

    def params(self):
        return [self.w, self.b] if self.b is not None else [self.w]

    def f(self, x):
        res = autodiff.dot(x, self.w)
        if self.b is not None:
            res += self.b
        return res


def LinearWithWeights(w: Tensor, b: Tensor | None) -> Linear:
    if b is not None:
        assert b.dim()[0] == w.dim()[1], "weight dim [a,b] must match bias dim [b]"
    return Linear(w=w, b=b)


class Sigmoid(Module):
    def f(self, x):
        return f32(1.0) / (f32(1.0) + (-x).exp())


class ReLU(Module):
    def f(self, x):
        return x * x.more_than(autodiff.constant(0.0, x.dim()))


class Softmax(Module):
    def __init__(self, dim):
        self.dim = dim

    def f(self, x):
        return x.exp() / x.exp().sum(self.dim)


class RMS(Module):
    def __init__(self, d_model):
        self.scale = autodiff.ones([d_model])

    def params(self):
        return [self.scale]

    def f(self, x):
        eps = f32(1e-9)
        var = x.pow2().mean(-1).unsqueeze(-1) + eps
        return self.scale * (x / var.sqrt())


class LayerNorm(Module):
    def __init__(self, d_model):
        self.scale = autodiff.ones([d_model])
        self.bias = autodiff.zeros([d_model])

    def params(self):
        return [self.scale]

    def f(self, x):
        eps = f32(1e-9)
        y = (x - x.mean(-1).unsqueeze(-1)) / (x.var(-1, 0) + eps).sqrt().unsqueeze(-1)
        return y * self.scale + self.bias


class ResidualRMS(Module):
    """RMS norm with the residual's addition in the same pass: `f(x, residual)` gives (y, h) with h = x + residual, the
    next layer's residual.  (`RMS` above is upstream's composition, src/nn/norm/rms.rs.)"""

    def __init__(self, d_model, eps=1e-6):
        self.scale = autodiff.ones([d_model])
        self.eps = eps

    def params(self):
        return [self.scale]

    def f(self, x, residual=None):
        return autodiff.rms_norm(x, self.scale, residual, self.eps)


class Rotary(Module):
    """Rotary positions for heads whose first `rot` elements are turned: pair i turns by base^(-2 i / rot) radians per
    position, worked out here in float64 and handed over in whole turns as two floats.

    For contexts longer than the one trained on, `stretch` divides the frequencies.  With `blend = (slow, fast, trained)`
    only slow pairs are stretched: those that make fewer than `slow` turns over `trained` positions wholly, those that
    make more than `fast` not at all, those between in proportion.  `gain` multiplies the turned elements."""

    def __init__(self, rot, base=10000.0, stretch=1.0, blend=None, interleaved=False, gain=1.0):
        if rot < 2 or rot % 2:
            raise ValueError("Rotary: an even number of elements is turned")
        if not (base > 0 and stretch > 0):
            raise ValueError("Rotary: base and stretch must be positive")
        turns = float(base) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot) / (2 * np.pi)
        part = np.ones_like(turns)
        if blend is not None:
            slow, fast, trained = blend
            if not 0 <= slow < fast:
                raise ValueError("Rotary: blend needs slow < fast")
            part = 1.0 - np.clip((turns * trained - slow) / (fast - slow), 0.0, 1.0)
        turns = turns * (part / stretch + (1.0 - part))
        hi = turns.astype(f32)
        self.table = np.stack([hi, (turns - hi).astype(f32)])
        self.interleaved, self.gain = interleaved, gain

    def f(self, x, positions=None, offset=0):
        table = autodiff.Value.new(self.table.reshape(-1), list(self.table.shape)).to_node()
        return autodiff.rotary(x, table, positions, offset, self.interleaved, self.gain)


class SelfAttention(Module):
    """Projections, rotary positions (when `rotary` is given) and attention of x [batch, tokens, d_model] to itself;
    `masks` are the keyword arguments of `autodiff.attention`."""

    def __init__(self, d_model, heads, kv_heads=None, rotary=None, rng=None, **masks):
        kv_heads = heads if kv_heads is None else kv_heads
        if d_model % heads or heads % kv_heads:
            raise ValueError("SelfAttention: d_model must be a multiple of heads, heads of kv_heads")
        self.heads, self.kv_heads, self.size = heads, kv_heads, d_model // heads
        s = f32(1.0 / np.sqrt(d_model))
        rng = rng or np.random.default_rng()

        def linear(inp, out):
            return Linear(w=autodiff.tensor(s * rng.standard_normal(inp * out, dtype=f32), [inp, out]))

        self.q, self.k, self.v = (linear(d_model, n * self.size) for n in (heads, kv_heads, kv_heads))
        self.o = linear(d_model, d_model)
        self.rotary, self.masks = rotary, masks

    def params(self):
        return [p for m in (self.q, self.k, self.v, self.o) for p in m.params()]

    def f(self, x, **masks):
        b, t, d = x.dim()
        flat = x.view([b * t, d])
        q = self.q.f(flat).view([b, t, self.heads, self.size])
        k = self.k.f(flat).view([b, t, self.kv_heads, self.size])
        v = self.v.f(flat).view([b, t, self.kv_heads, self.size])
        if self.rotary is not None:
            q, k = self.rotary.f(q), self.rotary.f(k)
        out = autodiff.attention(q, k, v, **{**self.masks, **masks})
        return self.o.f(out.view([b * t, d])).view([b, t, d])


def mse_loss(y: Tensor, target: Tensor) -> Tensor:
    """mean((y - target)^2) over every element, as a [1]-shaped tensor: the composition the reference's examples
    spell out by hand (`MSE` is on its to-do list, TODO.md:12): square, sum the axes from the last to the first,
    scale by the host-computed 1 / count."""
    d = y - target
    count = int(np.prod(d.dim()))
    s = d.pow2()
    while len(s.dim()) > 1:
        s = s.sum(len(s.dim()) - 1)
    return s.sum(0) * f32(1.0 / count)


class MSELoss(Module):
    def f(self, x: Tensor, target: Tensor = None) -> Tensor:
        return mse_loss(x, target)


class Sequential(Module):
    def __init__(self):
        self.n: list[Module] = []

    def insert(self, m: Module):
        self.n.append(m)

    def params(self):
        out = []
        for m in self.n:
            out.extend(m.params())
        return out

    def f(self, x):
        for m in self.n:
            x = m.f(x)
        return x


class SGD:
    """`p -= lr * p.grad(); p.forward()` per parameter (src/nn/optimizers/sgd.rs:9-14)."""

    def __init__(self, params, lr):
        self.n = list(params)
        self.lr = f32(lr)

    def step(self):
        for p in self.n:
            p -= self.lr * p.grad().to_node()
            p.forward()

    def zero_grad(self):
        for p in self.n:
            p.reset_grad()
