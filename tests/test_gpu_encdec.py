"""Cross attention and relative position bias against the fp64 oracle (MI355X).

Tolerances, per element, from the oracle's own values. u is half a step of the
type: 2^-8 (bf16), 2^-11 (fp16), 2^-24 (float32). Logits are fp32 sums of D
products and a bias, taken to exponents: their error is at most e = (D + 16)
2^-24 max(|scale| |q| |k| + |bias|), which moves a weight by the factor e^2e at
most (its own and the sum's), beside the exponential's 2^-21.
  O: the weights P round to the type (16 bits), then O does:
     u |O| + (u + 2 e + 2^-20) P |V|; fp16 weights below 2^-14 of the largest
     round to a grid of 2^-24: n 2^-24 max |V| more.
  dV: u |dV| + (u + 2 e + 2^-20) P^T |dO|
  dS = P (dP - D) rounds to the type as well; its fp32 dP and D = rowsum(dO O)
     are off by D 2^-23 of their magnitudes; with the given O:
     dQ: u |dQ| + (u + 2 e + 2^-19 + D 2^-23) |scale| P (|dP| + |D|) |K|, and dK;
     the same factor on sums of P (|dP| + |D|) by bucket for dT, without its
     rounding to 16 bits but with the fp32 sums' (2^-18).
"""
import math

import numpy as np
import pytest
import torch

import cuda_llm
import oracle
from _util import to_np

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "fp32"}


class Problem:
    """Inputs of one call and their oracle. junk: what lies past the lengths."""

    def __init__(self, dev, dtype, b, hq, hkv, sq, skv, d, lens=None, buckets=0, distance=128, causal=False,
                 scale=None, junk=None, seed=0, table=None, at_end=False, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.scale, self.causal, self.distance = dtype, scale, causal, distance
        self.lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
        self.n = [skv] * b if lens is None else [min(max(x, 0), skv) for x in lens]
        self.q = (torch.randn(b, hq, sq, d, generator=g) * magnitude).to(dtype).to(dev)
        self.k, self.v = (torch.randn(b, hkv, skv, d, generator=g).to(dtype).to(dev) for _ in range(2))
        self.dout = torch.randn(b, hq, sq, d, generator=g).to(dtype).to(dev)
        self.table = None
        if table is not None:
            self.table = table.to(dev)
        elif buckets:
            self.table = (2 * torch.randn(buckets, hq, generator=g)).to(dtype).to(dev)
        self.s = 1 / math.sqrt(d) if scale is None else scale
        kz, vz = to_np(self.k).copy(), to_np(self.v).copy()
        for i, n in enumerate(self.n):
            kz[i, :, n:], vz[i, :, n:] = 0, 0
            if junk is not None:
                self.k[i, :, n:], self.v[i, :, n:] = junk, junk
        self.np = dict(q=to_np(self.q), k=kz, v=vz, dout=to_np(self.dout))
        t = None if self.table is None else to_np(self.table)
        self.fwd = oracle.encdec_attention(self.np["q"], kz, vz, self.n, self.s, t, distance, causal, at_end)
        qk = np.abs(self.np["q"]).max() * np.abs(kz).max(initial=0)
        bias = 0 if t is None else np.abs(np.where(np.isfinite(t), np.clip(t, -32768, 32768), 0)).max()
        # (|q.k| is at most the largest row norms' product)
        qn = np.linalg.norm(self.np["q"], axis=-1).max(initial=0) * np.linalg.norm(kz, axis=-1).max(initial=0)
        self.e = (d + 16) * 2.0 ** -24 * (abs(self.s) * min(qn, d * qk) + bias)
        self.d = d

    def args(self):
        return (self.q, self.k, self.v) + (() if self.table is None else (self.table,))

    def kw(self):
        kw = dict(kv_lens=self.lens, softmax_scale=self.scale)
        if self.table is not None:
            kw.update(is_causal=self.causal, max_distance=self.distance)
        return kw

    def f(self, name):
        return getattr(cuda_llm, ("cross_attention" if self.table is None else "relative_bias_attention") + name)

    def check_out(self, out, what="out"):
        assert out.dtype == self.dtype and out.shape == self.q.shape
        near(out, self.fwd["out"], self.tol_out(), what)

    def tol_out(self):
        u, ref = U[self.dtype], self.fwd["out"]
        g = self.q.shape[1] // self.k.shape[1]
        pv = np.einsum("bhij,bhjd->bhid", self.fwd["p"], np.repeat(np.abs(self.np["v"]), g, axis=1))
        tol = u * np.abs(ref) + (u + 2 * self.e + 2.0 ** -20) * pv + 1e-30
        if self.dtype == torch.float16:
            tol += max(self.n) * 2.0 ** -24 * np.abs(self.np["v"]).max(initial=0) + 2.0 ** -25
        return tol

    def check_lse(self, lse):
        ref = self.fwd["lse"]
        assert lse.dtype == torch.float32
        x = to_np(lse).astype(np.float64)
        assert (np.isneginf(x) == np.isneginf(ref)).all()
        ok = np.isfinite(ref)
        near(x[ok], ref[ok], self.e + 2.0 ** -19 + 2.0 ** -22 * np.abs(ref[ok]), "lse")

    def check_grads(self, grads, out=None):
        """out: the output that the backward was given (None: its own forward's,
        rounded to the type, whose error D takes on)."""
        nb = 0 if self.table is None else self.table.shape[0]
        a = (self.np["q"], self.np["k"], self.np["v"], self.np["dout"], self.fwd, self.n, self.s, nb)
        o = None if out is None else to_np(out)
        ref = oracle.encdec_backward(*a, out=o)
        mag = oracle.encdec_backward(*a, out=o, magnitude=True)
        u = U[self.dtype]
        f = u + 2 * self.e + 2.0 ** -19 + self.d * 2.0 ** -23
        if out is None:
            f += 2 * u   # O's rounding and its weights', in D
        for name, t in zip(("dq", "dk", "dv", "dtable"), grads):
            assert t.dtype == self.dtype
            factor = f + (2.0 ** -18 if name == "dtable" else 0)
            tol = u * np.abs(ref[name]) + factor * mag[name] + 1e-30
            if self.dtype == torch.float16:
                # a dS or P below fp16's normal numbers: half a step of 2^-24
                # each, of up to as many terms
                big = max(np.abs(x).max(initial=0) for x in self.np.values())
                tol = tol + 2.0 ** -25 + max(max(self.n, default=0), self.q.shape[2] * self.q.shape[1]
                                             // self.k.shape[1]) * 2.0 ** -25 * big * max(1, abs(self.s))
            near(t, ref[name], tol, name)


def near(x, ref, tol, what):
    x = x if isinstance(x, np.ndarray) else x.detach().double().cpu().numpy()
    assert np.isfinite(x).all(), f"{what}: not finite"
    err = np.abs(x - ref) - tol
    if err.size and err.max() > 0:
        i = np.unravel_index(err.argmax(), err.shape)
        raise AssertionError(f"{what}{list(i)}: {x[i]} against {ref[i]}, tolerance {np.broadcast_to(tol, ref.shape)[i]:.3e}")


# (b, hq, hkv, sq, skv, lens)
CROSS = [
    (1, 1, 1, 1, 1, None),
    (2, 4, 2, 1, 333, [333, 40]),
    (3, 8, 2, 3, 65, [0, 64, 65]),
    (2, 4, 4, 33, 17, [1, 17]),
    (2, 3, 1, 100, 257, [257, 129]),
    (1, 2, 2, 300, 1000, None),
    (2, 32, 8, 50, 700, [700, 31]),
    (1, 4, 1, 520, 96, [-3]),
    (2, 2, 1, 257, 128, [500, 64]),
    (1, 16, 1, 5, 1500, [1499]),
]


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,sq,skv,lens", CROSS)
def test_cross_forward(dev, dtype, d, b, hq, hkv, sq, skv, lens):
    p = Problem(dev, dtype, b, hq, hkv, sq, skv, d, lens, junk=float("nan"))
    p.check_out(p.f("_forward")(*p.args(), **p.kw()))
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    p.check_out(out, "out with lse")
    p.check_lse(lse)


# (b, hq, hkv, sq, skv, lens, buckets, distance, causal)
BIAS = [
    (1, 1, 1, 1, 1, None, 4, 20, False),
    (1, 2, 2, 100, 100, None, 32, 128, False),
    (2, 4, 2, 100, 100, [100, 31], 32, 128, True),
    (3, 2, 2, 65, 65, [0, 64, 65], 10, 20, False),
    (1, 4, 4, 300, 300, [277], 64, 500, True),
    (2, 2, 1, 257, 257, [257, 40], 32, 20, False),
    (1, 3, 1, 513, 513, None, 8, 2000, False),
    (1, 2, 1, 700, 700, None, 256, 2048, True),
    (1, 2, 2, 90, 40, None, 32, 128, False),
    (1, 2, 1, 40, 390, None, 32, 128, False),
    (1, 2, 1, 40, 390, None, 6, 30, True),
    (2, 1, 1, 1100, 1100, [1100, 500], 32, 128, True),
    (2, 2, 1, 150, 150, [150, 99], 64, 20, True),
    (1, 2, 2, 150, 150, [143], 64, 9, False),
]


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,sq,skv,lens,buckets,distance,causal", BIAS)
def test_bias_forward(dev, dtype, d, b, hq, hkv, sq, skv, lens, buckets, distance, causal):
    p = Problem(dev, dtype, b, hq, hkv, sq, skv, d, lens, buckets, distance, causal, junk=float("nan"))
    p.check_out(p.f("_forward")(*p.args(), **p.kw()))
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    p.check_out(out, "out with lse")
    p.check_lse(lse)


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,sq,skv,lens", CROSS)
def test_cross_backward(dev, dtype, d, b, hq, hkv, sq, skv, lens):
    p = Problem(dev, dtype, b, hq, hkv, sq, skv, d, lens, junk=float("nan"))
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    grads = p.f("_backward")(p.dout, *p.args(), out, lse, **p.kw())
    p.check_grads(grads, out)


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,sq,skv,lens,buckets,distance,causal", BIAS)
def test_bias_backward(dev, dtype, d, b, hq, hkv, sq, skv, lens, buckets, distance, causal):
    p = Problem(dev, dtype, b, hq, hkv, sq, skv, d, lens, buckets, distance, causal, junk=float("nan"))
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    q, k, v, table = p.args()
    grads = p.f("_backward")(p.dout, q, k, v, out, lse, table, **p.kw())
    p.check_grads(grads, out)


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,s,lens,buckets,distance", [
    (1, 1, 1, 1, None, 2, 8),
    (3, 4, 2, 100, [1, 0, 100], 32, 128),
    (2, 32, 8, 1000, [1000, 333], 32, 128),
    (2, 40, 2, 300, [299, 17], 64, 500),
    (1, 2, 2, 3000, None, 256, 2048),
    (2, 4, 1, 500, [500, 36], 64, 20),
    (4, 8, 8, 700, [700, 500, 130, 16], 10, 20),
])
def test_bias_decode(dev, dtype, d, b, hq, hkv, s, lens, buckets, distance):
    p = Problem(dev, dtype, b, hq, hkv, 1, s, d, lens, buckets, distance, True, junk=float("nan"), at_end=True)
    q, k, v, table = p.args()
    p.check_out(cuda_llm.relative_bias_decode(q, k, v, table, p.lens, max_distance=distance))
