"""Cross attention and relative position bias at the edges (MI355X): masks and
tables that leave nothing, scales, sizes past 32 bits, orders of many sequences,
the forms of a call (module and general path, streams, graphs), and the operators
together. Tolerances as in test_gpu_encdec.py, or derived where they are used.
"""
import math

import numpy as np
import pytest
import torch

import cuda_amd._lib as L
import cuda_amd.api as api
import cuda_llm
import oracle
from _util import to_np
from test_gpu_encdec import DT, IDS, Problem, U, near

pytestmark = pytest.mark.gpu
INF = float("inf")


def _all(p):
    """Forward, forward with LSE and backward of a Problem against the oracle."""
    p.check_out(p.f("_forward")(*p.args(), **p.kw()))
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    p.check_out(out, "out with lse")
    p.check_lse(lse)
    grads = p.f("_backward")(p.dout, *p.args()[:3], out, lse, *p.args()[3:], **p.kw())
    p.check_grads(grads, out)
    return [out, lse, *grads]


def _equal(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


# ---------------------------------------------------------------------------
# Values
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-12, 3.0])
@pytest.mark.parametrize("buckets", [0, 32])
def test_scales(dev, dtype, d, scale, buckets):
    _all(Problem(dev, dtype, 2, 4, 2, 70, 150, d, [150, 33], buckets, 64, scale=scale, junk=INF, magnitude=0.5))


# which entries of the table (8 buckets, 4 of a side, 2 heads) get `value`
TABLES = {
    "all": lambda t, v: t.fill_(v),
    "one head": lambda t, v: t[:, 1].fill_(v),
    "own token": lambda t, v: t[0].fill_(v),
    "far": lambda t, v: (t[3].fill_(v), t[7:].fill_(v)),
    "near": lambda t, v: (t[:3].fill_(v), t[5:7].fill_(v)),
    "after": lambda t, v: t[4:].fill_(v),
    "before": lambda t, v: t[:4].fill_(v),
}


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", TABLES)
@pytest.mark.parametrize("value", [-INF, "lowest"])
@pytest.mark.parametrize("causal", [False, True])
def test_masking_tables(dev, dtype, d, where, value, causal):
    """Entries of -inf (rows may be left without a key: zeros, LSE -inf, no
    gradient) and of the type's lowest number (clamped: where every key has it,
    all count alike)."""
    value = torch.finfo(dtype).min if value == "lowest" else value
    t = torch.randn(4 if causal else 8, 2, generator=torch.Generator().manual_seed(3)).to(dtype)
    TABLES[where](t, value)
    p = Problem(dev, dtype, 2, 2, 1, 140, 140, d, [140, 70], buckets=t.shape[0], distance=40, causal=causal, table=t,
                junk=float("nan"))
    # (against the clamp, logits of 2^15 have steps of 2^-8: inputs that small
    # steps of them do not show)
    if value != -INF:
        p.e += 2.0 ** -8
    _all(p)


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("table_dtype", DT, ids=IDS.get)
def test_table_types(dev, dtype, table_dtype):
    t = torch.randn(16, 4, generator=torch.Generator().manual_seed(5)).to(table_dtype)
    p = Problem(dev, dtype, 1, 4, 2, 80, 80, 64, buckets=16, distance=30, table=t)
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    p.check_out(out)
    q, k, v, table = p.args()
    grads = p.f("_backward")(p.dout, q, k, v, out, lse, table, **p.kw())
    assert grads[3].dtype == table_dtype
    ref = oracle.encdec_backward(p.np["q"], p.np["k"], p.np["v"], p.np["dout"], p.fwd, p.n, p.s, 16, out=to_np(out))
    mag = oracle.encdec_backward(p.np["q"], p.np["k"], p.np["v"], p.np["dout"], p.fwd, p.n, p.s, 16, out=to_np(out),
                                 magnitude=True)
    near(grads[3], ref["dtable"], U[table_dtype] * np.abs(ref["dtable"]) + (
        U[dtype] + 2 * p.e + 2.0 ** -17 + 64 * 2.0 ** -23) * mag["dtable"], "dtable")
    dq = Problem(dev, dtype, 2, 4, 2, 1, 90, 64, [90, 1], 16, 30, True, table=t, at_end=True)
    dq.check_out(cuda_llm.relative_bias_decode(*dq.args(), dq.lens, max_distance=30))


STARTS = [([0], True), ([0], False), ([0, 0, 0], False), ([0, 0, 5, 5], True), ([0, 3, 3, 40], False),
          ([0, 2048], True), ([0, 2048], False), (list(range(0, 128)), False), (list(range(0, 256)), True)]


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("starts,causal", STARTS, ids=[f"{len(s)}-{s[-1]}-{c}" for s, c in STARTS])
def test_bucket_lists(dev, monkeypatch, dtype, d, starts, causal):
    """Any list of first distances: one bucket, empty ones, as many as there may be."""
    import ctypes
    array = (ctypes.c_int32 * len(starts))(*starts)
    monkeypatch.setattr(api, "_bucket_starts", lambda *a: (array, ctypes.addressof(array)))

    def bucket(distance, num_buckets, is_causal, max_distance):
        n = max(-distance, 0) if is_causal else abs(distance)
        return max(i for i, s in enumerate(starts) if s <= n) + (len(starts) if distance > 0 and not is_causal else 0)

    monkeypatch.setattr(oracle.encdec, "relative_bucket", bucket)
    nb = len(starts) if causal else 2 * len(starts)
    _all(Problem(dev, dtype, 2, 4, 2, 130, 130, d, [130, 77], nb, causal=causal, junk=float("nan")))
    if causal:
        p = Problem(dev, dtype, 2, 4, 2, 1, 300, d, [300, 9], nb, causal=True, at_end=True, junk=float("nan"))
        p.check_out(cuda_llm.relative_bias_decode(*p.args(), p.lens))


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("buckets", [0, 32])
def test_nan_stays_in_its_head_and_row(dev, dtype, buckets):
    """A NaN in one query, or among one head's keys, leaves all other rows and
    heads as they are."""
    p = Problem(dev, dtype, 2, 4, 2, 70, 200, 64, [200, 90], buckets)
    ref = p.f("_forward")(*p.args(), **p.kw()).clone()
    keep = p.q.clone()
    p.q[1, 2, 33] = float("nan")
    out = p.f("_forward")(*p.args(), **p.kw())
    same = torch.ones(2, 4, 70, dtype=torch.bool, device=dev)
    same[1, 2, 33] = False
    assert torch.equal(out[same], ref[same])
    p.q.copy_(keep)
    p.k[0, 1, 7] = float("nan")
    out = p.f("_forward")(*p.args(), **p.kw())
    assert torch.equal(out[0, :2], ref[0, :2]) and torch.equal(out[1], ref[1])


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("magnitude", [30.0, 300.0])
def test_sharp_rows(dev, dtype, magnitude):
    """Logits far apart: rising and falling along the keys, so that tiles at the
    start or the end of the walk take no part."""
    for sign in (1, -1):
        p = Problem(dev, dtype, 1, 2, 2, 40, 500, 64, [490], scale=1.0)
        ramp = torch.linspace(0, magnitude, 500, device=dev) * sign
        p.q.zero_()
        p.q[..., 0] = 1
        p.k[..., 0] = ramp.to(dtype)
        p.np["q"], p.np["k"] = to_np(p.q), to_np(p.k)
        p.np["k"][:, :, 490:] = 0
        p.fwd = oracle.encdec_attention(p.np["q"], p.np["k"], p.np["v"], p.n, 1.0)
        p.e = 80 * 2.0 ** -24 * magnitude
        _all(p)


# ---------------------------------------------------------------------------
# Sizes and orders
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("b,hq,hkv", [(70, 8, 2), (64, 8, 8), (5, 24, 3), (7, 12, 4), (9, 1, 1)])
@pytest.mark.parametrize("buckets", [0, 16])
def test_many_sequences(dev, dtype, b, hq, hkv, buckets):
    """Sequences ranked by length, past 64 of them, and heads that 8 does not divide."""
    lens = [(37 * i * i + 11) % 91 for i in range(b)]
    lens[b // 2], lens[b // 3] = 0, 200
    _all(Problem(dev, dtype, b, hq, hkv, 40, 90, 64, lens, buckets, 30, junk=float("nan")))


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("buckets", [0, 32])
def test_split_walks(dev, dtype, d, buckets):
    """Few rows over many keys (the walk in parts), some of them without a key."""
    _all(Problem(dev, dtype, 3, 2, 1, 40, 2500, d, [2500, 0, 70], buckets, junk=float("nan")))
    _all(Problem(dev, dtype, 1, 1, 1, 1, 4099, d, None, buckets))


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,s", [(1, 1, 1, 64), (1, 1, 1, 65), (3, 24, 2, 700), (2, 4, 4, 5000), (1, 16, 1, 20000)])
def test_steps_in_any_workspace(dev, dtype, d, b, hq, hkv, s):
    """The step's walk in as many parts as the workspace holds: from the least to
    more than its query asks, through the C ABI."""
    lens = [s, s // 3, 0][:b]
    p = Problem(dev, dtype, b, hq, hkv, 1, s, d, lens, 32, 128, True, at_end=True, junk=float("nan"))
    starts = api._bucket_starts(32, True, 128)[0]
    dt = api._DT[dtype]
    least = L.load().ca_decode_workspace_bytes(b, hq, d, s)
    best = L.load().ca_relative_bias_decode_workspace_bytes(dt, b, hq, hkv, s, d)
    for nbytes in sorted({least, (least + best) // 32 * 16, best, best + 4096}):
        ws = torch.full((max(nbytes, 16),), 255, dtype=torch.uint8, device=dev)
        out = torch.full_like(p.q, float("nan"))
        L.call("ca_relative_bias_decode", dt, *(api._ptr(t) for t in (p.q, p.k, p.v, p.table)), api._DT[p.table.dtype],
               starts, 32, api._ptr(p.lens), api._ptr(out), b, hq, hkv, s, d, p.s, api._ptr(ws), nbytes, api._stream())
        p.check_out(out, f"{nbytes} bytes")
    c = Problem(dev, dtype, b, hq, hkv, 1, s, d, lens, junk=float("nan"))
    c.check_out(cuda_llm.cross_attention(*c.args(), **c.kw()))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,sq,skv,lens", [
    (1, 8, 8, 64, 4000, None), (2, 8, 2, 17, 3001, [3001, 5]), (1, 32, 8, 20, 2500, [0]), (1, 3, 1, 85, 5000, [4999])])
def test_few_float32_rows(dev, d, b, hq, hkv, sq, skv, lens):
    """Up to 256 rows of a kv head that the step's walk takes, and as tiles (with an LSE)."""
    _all(Problem(dev, torch.float32, b, hq, hkv, sq, skv, d, lens, junk=float("nan")))


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
def test_empty_sizes(dev, dtype):
    new = lambda *s: torch.randn(*s, device=dev).to(dtype)
    table = new(8, 4)
    for b, sq, skv in ((0, 5, 7), (2, 0, 7), (2, 5, 0), (0, 0, 0)):
        q, k, v = new(b, 4, sq, 64), new(b, 2, skv, 64), new(b, 2, skv, 64)
        for name, t, kw in (("cross_attention", (), {}), ("relative_bias_attention", (table,), dict(max_distance=20))):
            f = lambda suffix: getattr(cuda_llm, name + suffix)
            out, lse = f("_forward_lse")(q, k, v, *t, **kw)
            assert out.shape == q.shape and not out.any() and torch.isneginf(lse).all()
            assert not f("_forward")(q, k, v, *t, **kw).any()
            grads = f("_backward")(torch.randn_like(q), q, k, v, out, lse, *t, **kw)
            for g, x in zip(grads, (q, k, v, *t)):
                assert g.shape == x.shape and g.dtype == x.dtype and not g.any()
    for b, skv in ((0, 9), (2, 0)):
        out = cuda_llm.relative_bias_decode(new(b, 4, 1, 64), new(b, 2, skv, 64), new(b, 2, skv, 64), table,
                                            max_distance=20)
        assert out.shape == (b, 4, 1, 64) and not out.any()


class _Slice(Problem):
    """A Problem of some heads of a call's tensors."""

    def __init__(self, q, k, v, dout, table=None, scale=None, causal=False, distance=128, at_end=False):
        self.q, self.k, self.v, self.dout, self.table = q, k, v, dout, table
        self.dtype, self.d, self.scale, self.causal, self.distance = q.dtype, q.shape[3], scale, causal, distance
        self.n = [k.shape[2]] * q.shape[0]
        self.s = 1 / math.sqrt(self.d) if scale is None else scale
        self.np = dict(q=to_np(q), k=to_np(k), v=to_np(v), dout=to_np(dout))
        t = None if table is None else to_np(table)
        self.fwd = oracle.encdec_attention(self.np["q"], self.np["k"], self.np["v"], self.n, self.s, t, distance,
                                           causal, at_end)
        norm = lambda x: np.linalg.norm(x, axis=-1).max()
        self.e = (self.d + 16) * 2.0 ** -24 * (abs(self.s) * norm(self.np["q"]) * norm(self.np["k"]) + (
            0 if t is None else np.abs(t).max()))


@pytest.mark.parametrize("sq", [1, 33])
def test_keys_past_32_bits(dev, sq):
    """k and v of 2.6e9 elements each: the last heads, forward, decode, backward."""
    h, s, d = 1024, 20000, 128
    g = torch.Generator(device=dev).manual_seed(1)
    q, dout = (torch.randn(1, h, sq, d, device=dev, dtype=torch.bfloat16, generator=g) for _ in range(2))
    k, v = (torch.randn(1, h, s, d, device=dev, dtype=torch.bfloat16, generator=g) for _ in range(2))
    table = torch.randn(32, h, device=dev, generator=g).to(torch.bfloat16)
    last = lambda *t: [x[:, -2:].contiguous() for x in t]
    p = _Slice(*last(q, k, v, dout))
    out, lse = cuda_llm.cross_attention_forward_lse(q, k, v)
    p.check_out(out[:, -2:])
    p.check_lse(lse[:, -2:])
    grads = cuda_llm.cross_attention_backward(dout, q, k, v, out, lse)
    p.check_grads([x[:, -2:] for x in grads], out[:, -2:])
    del grads
    _Slice(*last(q, k, v, dout)).check_out(cuda_llm.cross_attention(q, k, v)[:, -2:])
    if sq == 1:
        one = cuda_llm.relative_bias_decode(q, k, v, table)
        _Slice(*last(q, k, v, dout, ), table[:, -2:].contiguous(), causal=True, at_end=True).check_out(one[:, -2:])


@pytest.mark.parametrize("bias", [False, True])
def test_queries_past_32_bits(dev, bias):
    """q of 2.6e9 elements: the last heads of out, lse and dq."""
    h, s, n, d = 1024, 20000, 100, 128
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn(1, h, s, d, device=dev, dtype=torch.bfloat16, generator=g)
    k, v = (torch.randn(1, h, n, d, device=dev, dtype=torch.bfloat16, generator=g) for _ in range(2))
    dout = torch.randn(1, 1, s, d, device=dev, dtype=torch.bfloat16, generator=g).expand(1, h, s, d).contiguous()
    table = torch.randn(32, h, device=dev, generator=g).to(torch.bfloat16) if bias else None
    last = [x[:, -1:].contiguous() for x in (q, k, v, dout)]
    p = _Slice(*last, table[:, -1:].contiguous() if bias else None)
    t, kw = ((table,), dict(max_distance=128)) if bias else ((), {})
    out, lse = p.f("_forward_lse")(q, k, v, *t, **kw)
    p.check_out(out[:, -1:])
    p.check_lse(lse[:, -1:])
    grads = p.f("_backward")(dout, q, k, v, out, lse, *t, **kw)
    p.check_grads([x[:, -1:] for x in grads], out[:, -1:])


def test_shared_head_queries_past_32_bits(dev):
    """The rows of a kv head's 32 query heads, 2.6e9 elements one after the other."""
    h, s, n, d = 32, 640000, 64, 128
    g = torch.Generator(device=dev).manual_seed(1)
    q, dout = (torch.randn(1, h, s, d, device=dev, dtype=torch.bfloat16, generator=g) for _ in range(2))
    k, v = (torch.randn(1, 1, n, d, device=dev, dtype=torch.bfloat16, generator=g) for _ in range(2))
    out, lse = cuda_llm.cross_attention_forward_lse(q, k, v)
    dq = cuda_llm.cross_attention_backward(dout, q, k, v, out, lse)[0]
    last = lambda t: t[:, -1:, -1000:].contiguous()
    p = _Slice(last(q), k, v, last(dout))
    p.check_out(last(out))
    p.check_lse(last(lse))
    p.check_grads([last(dq)], last(out))


# ---------------------------------------------------------------------------
# The forms of a call
# ---------------------------------------------------------------------------
@pytest.fixture
def general(monkeypatch):
    """Calls f through the general path."""
    def run(f):
        with monkeypatch.context() as m:
            m.setattr(api, "_native_module", L._General())
            m.setattr(api, "_native", lambda: api._native_module)
            return f()
    return run


def _calls(p):
    """Every result of the operator of a Problem."""
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    grads = p.f("_backward")(p.dout, *p.args()[:3], out, lse, *p.args()[3:], **p.kw())
    return [p.f("_forward")(*p.args(), **p.kw()), out, lse, *grads]


def _shift(t):
    """The same values, contiguous, one element past a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:] = t.flatten()
    return buf[1:].view(t.shape)


FORMS = [dict(b=2, hq=4, hkv=2, sq=100, skv=130, d=64, lens=[130, 7]), dict(b=1, hq=8, hkv=8, sq=3, skv=700, d=128),
         dict(b=2, hq=4, hkv=4, sq=90, skv=90, d=64, lens=[60, 90], buckets=32),
         dict(b=1, hq=2, hkv=1, sq=200, skv=200, d=128, buckets=16, distance=40, causal=True)]


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_same_bytes_either_way(dev, general, dtype, form):
    p = Problem(dev, dtype, **FORMS[form])
    ref = _calls(p)
    _equal(ref, _calls(p))
    _equal(ref, general(lambda: _calls(p)))
    name = "cross_attention" if p.table is None else "relative_bias_attention"
    rest = () if p.table is None else (p.causal, None, api._starts_address(p.table, p.causal, p.distance))
    assert getattr(L.native(), name + "_forward")(*p.args(), p.lens, *(rest or (None,))) is not None
    if p.lens is not None:      # lengths as 64-bit integers, past either end
        lens = p.lens
        for big in (lens.long(), torch.where(lens == p.k.shape[2], 1 << 40, lens.long())):
            p.lens = big
            _equal(ref, _calls(p))
        for t in (torch.uint8, torch.int16):
            p.lens = lens.to(t)
            _equal(ref, _calls(p))
        p.lens = torch.stack([lens, lens], 1)[:, 0]   # a strided view
        _equal(ref, _calls(p))
        p.lens = lens
    for x in ("q", "k", "v", "dout"):   # off the 16-byte grid
        setattr(p, x, _shift(getattr(p, x)))
    _equal(ref, _calls(p))
    if p.table is not None:
        p.table = p.table.t().contiguous().t()   # strided
        _equal(ref, _calls(p))
        p.table = _shift(p.table)
        _equal(ref, _calls(p))


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
def test_decode_same_bytes_either_way(dev, general, dtype):
    p = Problem(dev, dtype, 3, 8, 2, 1, 300, 128, [300, 0, 17], 32, 128, True, at_end=True)
    f = lambda: [cuda_llm.relative_bias_decode(p.q, p.k, p.v, p.table, p.lens)]
    ref = f()
    _equal(ref, f())
    _equal(ref, general(f))
    p.lens = p.lens.long() + torch.tensor([1 << 35, 0, 0], device=dev)
    _equal(ref, f())
    p.q, p.k, p.v = _shift(p.q), _shift(p.k), _shift(p.v)
    _equal(ref, f())


def test_refusals(dev):
    new = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    q, k, table = new(2, 4, 5, 64), new(2, 2, 7, 64), new(8, 4)
    t = lambda x: x.transpose(1, 2)
    bad = [((t(new(2, 5, 4, 64)), k, k), "contiguous"), ((q, t(new(2, 7, 2, 64)), k), "contiguous"),
           ((q, k, new(2, 2, 8, 64)), "identical"), ((q, new(2, 3, 7, 64), new(2, 3, 7, 64)), "dividing"),
           ((q, new(1, 2, 7, 64), new(1, 2, 7, 64)), "batch"), ((q, k.half(), k.half()), "same dtype"),
           ((new(2, 4, 5, 32), new(2, 2, 7, 32), new(2, 2, 7, 32)), "head_dim"), ((q[0], k[0], k[0]), "4D"),
           ((q.double(), k.double(), k.double()), "type"), ((q, k.cpu(), k), "CUDA")]
    for args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.cross_attention(*args)
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.relative_bias_attention(*args, table, max_distance=20)
    for lens, word in ((torch.zeros(2), "device"), (new(3, dtype=torch.int32), "batch"), (new(2), "integers"),
                       (new(2, 1, dtype=torch.int32), "batch"), (new(2, dtype=torch.bool), "integers")):
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.cross_attention(q, k, k, lens)
    for tab, kw, word in ((new(8, 3), {}, "num_heads"), (new(8), {}, "num_buckets"), (new(7, 4), {}, "even"),
                          (new(8, 4, dtype=torch.int32), {}, "type"), (table.cpu(), {}, "device"),
                          (table, dict(max_distance=0), "max_distance"), (table, dict(max_distance=1 << 40), "max_distance"),
                          (new(258, 4), {}, "buckets"), (table, dict(max_distance=20.0), "integer")):
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.relative_bias_attention(q, k, k, tab, **kw)
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.relative_bias_attention_forward_lse(q, k, k, tab, **kw)
    with pytest.raises(RuntimeError, match="must be 1"):
        cuda_llm.relative_bias_decode(q, k, k, table, max_distance=20)
    with pytest.raises(RuntimeError, match="finite"):
        cuda_llm.cross_attention(q, k, k, None, math.nan)
    out, lse = cuda_llm.cross_attention_forward_lse(q, k, k)
    for args, word in (((out[:, :, :4], q, k, k, out, lse), "shape"), ((out, q, k, k, out, lse[:, :3]), "lse"),
                       ((out.half(), q, k, k, out, lse), "dtype"), ((out, q, k, k, out.cpu(), lse), "device")):
        with pytest.raises(RuntimeError, match=word):
            cuda_llm.cross_attention_backward(*args)


def test_streams(dev):
    """Two calls at once on two streams, neither of them the default one."""
    ps = [Problem(dev, torch.bfloat16, seed=i, **FORMS[i]) for i in range(4)]
    ref = [_calls(p) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st, p in zip(streams, ps):
            with torch.cuda.stream(st):
                got.append(_calls(p))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        _equal(ref[i % 4], x)


def _graph(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
def test_graphs(dev, dtype):
    """Captured calls, replayed in turn with new inputs and eager work between."""
    ps = [Problem(dev, dtype, seed=i, **f) for i, f in enumerate(FORMS)]
    step = Problem(dev, dtype, 2, 8, 2, 1, 900, 64, [900, 5], 32, 128, True, at_end=True)
    fs = [lambda p=p: _calls(p) for p in ps]
    fs.append(lambda: [cuda_llm.relative_bias_decode(step.q, step.k, step.v, step.table, step.lens)])
    graphs = [_graph(f) for f in fs]
    for r in range(4):
        for p in ps + [step]:
            for x in (p.q, p.k, p.v, p.dout):
                x.copy_(torch.randn(x.shape, device=dev))
            if p.lens is not None:
                p.lens.copy_(torch.randint(0, p.k.shape[2] + 1, p.lens.shape, device=dev))
            if p.table is not None:
                p.table.copy_(torch.randn(p.table.shape, device=dev))
        ref = [[x.clone() for x in f()] for f in fs]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, (_, b) in zip(ref, graphs):
            _equal(a, b)


def test_training_step_in_a_graph(dev):
    """Forward and backward through autograd, captured."""
    p = Problem(dev, torch.bfloat16, **FORMS[2])

    def step():
        leaves = [x.detach().requires_grad_() for x in p.args()]
        out = cuda_llm.relative_bias_attention(*leaves, p.lens)
        return [out.detach(), *torch.autograd.grad(out, leaves, p.dout)]

    g, got = _graph(step)
    for r in range(3):
        p.q.copy_(torch.randn(p.q.shape, device=dev))
        ref = [x.clone() for x in step()]
        g.replay()
        torch.cuda.synchronize()
        _equal(ref, got)


# ---------------------------------------------------------------------------
# Gradients
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("sq,skv", [(70, 96), (40, 3000), (1, 1)])
def test_what_the_rounding_took(dev, general, dtype, sq, skv):
    """Equal logits have weights of exactly 1, and sums of small whole numbers are
    exact: out and its rest are the mean to half a step of the type's square (a
    rest rounds to u of at most u |out|), float32's, and fp16's smallest number."""
    p = Problem(dev, dtype, 2, 2, 1, sq, skv, 64, [skv, (skv + 1) // 2], buckets=8, distance=20)
    p.q.zero_()
    p.table.zero_()
    p.v.copy_(torch.randint(-7, 8, p.v.shape, device=dev))
    address = api._starts_address(p.table, False, 20)
    out, lse, low = L.native().relative_bias_attention_forward_train(*p.args(), p.lens, False, None, address)
    _equal([out, lse], p.f("_forward_lse")(*p.args(), **p.kw()))
    _equal([out, lse, low], api._encdec_forward(*p.args()[:3], p.lens, None, True, (p.table, 20), False, True))
    for i, n in enumerate(p.n):
        ref = np.broadcast_to(to_np(p.v)[i, :, :n].astype(np.float64).mean(1, keepdims=True), (2, sq, 64))
        u = U[dtype]
        near(out[i].double() + low[i].double(), ref, (u * u + 2.0 ** -21) * np.abs(ref) + 2.0 ** -25 * (
            dtype == torch.float16) + 1e-30, "out + low")


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_autograd(dev, dtype, form):
    p = Problem(dev, dtype, **FORMS[form])
    leaves = [x.detach().clone().requires_grad_() for x in p.args()]
    # not contiguous, as an upstream transpose leaves it
    w = p.dout.transpose(1, 2).contiguous().transpose(1, 2)
    out = p.f("")(*leaves, **p.kw())
    p.check_out(out)
    p.check_grads(torch.autograd.grad(out, leaves, w))
    # one input alone
    for i, x in enumerate(p.args()):
        one = [y.detach() for y in p.args()]
        one[i] = x.detach().clone().requires_grad_()
        out = p.f("")(*one, **p.kw())
        (out.float() * p.dout.float()).sum().backward()
        assert one[i].grad.shape == x.shape
    with torch.no_grad():
        assert not p.f("")(*leaves, **p.kw()).requires_grad
    # a second derivative is refused
    out = p.f("")(*leaves, **p.kw())
    g, = torch.autograd.grad(out, leaves[:1], w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(dev, causal):
    """float32, the derivative of one output by one input number (by one bucket's
    value), against the four-point difference of step h = 2^-4. Its truncation is
    h^4 / 30 of the fifth derivative; a logit moves by at most |a| = 1 per unit
    here, and the fifth derivative of a softmax mean is at most 2^5 4! |a|^5 max
    |v| (each order multiplies by a deviation of at most 2 |a| and counts its
    factors); outputs are off by 2 e + 2^-19 of max |v|, 18 of them over 12 h."""
    p = Problem(dev, torch.float32, 1, 2, 1, 20, 20, 64, [17], 8, 12, causal, magnitude=0.5)
    q, k, v, table = p.args()
    assert float(max(q.abs().max(), k.abs().max())) * p.s <= 1
    out, lse = p.f("_forward_lse")(*p.args(), **p.kw())
    h = 2.0 ** -4
    vmax = float(v.abs().max())
    tol = (h ** 4 / 30 * 32 * 24 + 18 * (2 * p.e + 2.0 ** -19) / (12 * h)) * vmax + 1e-5
    assert tol < 0.05
    rng = np.random.default_rng(0)
    seen = 0.0
    for _ in range(12):
        head, row, c = rng.integers(2), rng.integers(20), rng.integers(64)
        dout = torch.zeros_like(out)
        dout[0, head, row, c] = 1
        grads = p.f("_backward")(dout, q, k, v, out, lse, table, **p.kw())
        key = rng.integers(min(row + 1, 17) if causal else 17)
        bucket = int(p.fwd["bucket"][0, row, key])
        for x, g, at in ((q, grads[0], (0, head, row, rng.integers(64))), (k, grads[1], (0, 0, key, rng.integers(64))),
                         (v, grads[2], (0, 0, key, c)), (table, grads[3], (bucket, head))):
            was = x[at].clone()
            f = []
            for m in (-2, -1, 1, 2):
                x[at] = was + m * h
                f.append(float(p.f("_forward")(*p.args(), **p.kw())[0, head, row, c]))
            x[at] = was
            diff = (8 * (f[2] - f[1]) - (f[3] - f[0])) / (12 * h)
            assert abs(diff - float(g[at])) <= tol
            seen = max(seen, abs(diff))
    assert seen > 10 * tol


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def _plain(q, k, v, lens, table=None, causal=False, distance=128, scale=1.0):
    """float64 on the CPU, differentiable."""
    x = q @ k.repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(2, 3) * scale
    n = k.shape[2]
    mask = (torch.arange(n)[None, :] >= torch.tensor(lens)[:, None])[:, None, None, :].expand(x.shape)
    if table is not None:
        ids = torch.tensor(oracle.bucket_matrix(q.shape[2], n, table.shape[0], causal, distance))
        x = x + table[ids].permute(2, 0, 1)
    if causal:
        mask = mask | torch.ones(n, n, dtype=torch.bool).triu(1)
    p = torch.softmax(x.masked_fill(mask, -math.inf), -1)
    return p @ v.repeat_interleave(q.shape[1] // k.shape[1], 1)


def _layer(x, y, w, tables, lens_x, lens_y, bias_op, cross_op, noise=lambda t: t):
    """A small encoder and decoder layer: x, y [B, S, H * 64]."""
    heads = lambda t, m: (t @ m).unflatten(-1, (-1, 64)).transpose(1, 2).contiguous()
    flat = lambda t: noise(t).transpose(1, 2).flatten(2)
    x = x + flat(bias_op(heads(x, w[0]), heads(x, w[1]), heads(x, w[2]), tables[0], lens_x, False))
    y = y + flat(bias_op(heads(y, w[3]), heads(y, w[4]), heads(y, w[5]), tables[1], lens_y, True))
    return y + flat(cross_op(heads(y, w[6]), heads(x, w[7]), heads(x, w[8]), lens_x))


def test_a_layer_of_all_three(dev):
    """Encoder self-attention, decoder self-attention and cross attention in
    training, float32 against float64. Every operator's results are within 2^-17
    of their size (test_gpu_encdec.py; the products' error is float32's as well);
    what that does to the layer is measured in float64, with results off by that
    much at random: 16 times the largest of 4 such changes is allowed."""
    b, h, sx, sy, lens_x, lens_y = 2, 2, 90, 70, [90, 41], [70, 33]
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float().double()
    x, y = rand(b, sx, h * 64), rand(b, sy, h * 64)
    w = [(rand(h * 64, h * 64) * 0.06).float().double() for _ in range(9)]
    tables = [rand(32, h), rand(16, h)]
    wout = rand(b, sy, h * 64)
    for i, n in enumerate(lens_y):
        wout[i, n:] = 0

    def run(bias_op, cross_op, to, lens_x, lens_y, noise=lambda t: t):
        leaves = [to(t).requires_grad_() for t in (x, y, *w, *tables)]
        out = _layer(leaves[0], leaves[1], leaves[2:11], leaves[11:], lens_x, lens_y, bias_op, cross_op, noise)
        grads = torch.autograd.grad((out * to(wout)).sum(), leaves)
        return [t.detach().double().cpu() for t in (out, *grads)]

    plain = (lambda q, k, v, t, n, c: _plain(q, k, v, n, t, c), lambda q, k, v, n: _plain(q, k, v, n, scale=0.125))
    ref = run(*plain, lambda t: t.clone(), lens_x, lens_y)
    spread = [torch.zeros_like(t) for t in ref]
    for _ in range(4):
        off = run(*plain, lambda t: t.clone(), lens_x, lens_y,
                  lambda t: t * (1 + 2.0 ** -17 * (2 * torch.rand(t.shape, generator=g, dtype=t.dtype) - 1)))
        spread = [torch.maximum(s, (a - r).abs().max().expand_as(s)) for s, a, r in zip(spread, off, ref)]
    nx, ny = (torch.tensor(n, dtype=torch.int32, device=dev) for n in (lens_x, lens_y))
    got = run(lambda q, k, v, t, n, c: cuda_llm.relative_bias_attention(q, k, v, t, n, c, 1.0),
              lambda q, k, v, n: cuda_llm.cross_attention(q, k, v, n), lambda t: t.float().to(dev), nx, ny)
    for i, (a, r, s) in enumerate(zip(got, ref, spread)):
        if i == 0:   # (rows past a sequence's end are its own business)
            keep = torch.arange(sy)[None, :] < torch.tensor(lens_y)[:, None]
            a, r, s = a[keep], r[keep], s[keep]
        near(a, r.numpy(), 16 * s.numpy(), f"result {i}")


@pytest.mark.parametrize("dtype", DT, ids=IDS.get)
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 8, 2)])
def test_token_by_token(dev, dtype, d, hq, hkv):
    """The decode step over a growing cache gives the rows of the causal call, and
    one query's cross attention those of all."""
    s = 150
    p = Problem(dev, dtype, 2, hq, hkv, s, s, d, None, 32, 100, True)
    c = Problem(dev, dtype, 2, hq, hkv, s, 333, d, [333, 20])
    kc, vc = (torch.full_like(t, float("nan")) for t in (p.k, p.v))
    tol, tol_c = p.tol_out(), c.tol_out()
    for i in range(s):
        kc[:, :, i], vc[:, :, i] = p.k[:, :, i], p.v[:, :, i]
        if i not in (0, 1, 15, 16, 17, 63, 64, 99, 100, 101, 148, 149):
            continue
        n = torch.full((2,), i + 1, dtype=torch.int32, device=dev)
        one = cuda_llm.relative_bias_decode(p.q[:, :, i:i + 1].contiguous(), kc, vc, p.table, n, max_distance=100)
        near(one, p.fwd["out"][:, :, i:i + 1], tol[:, :, i:i + 1], f"token {i}")
        one = cuda_llm.cross_attention(c.q[:, :, i:i + 1].contiguous(), c.k, c.v, c.lens)
        near(one, c.fwd["out"][:, :, i:i + 1], tol_c[:, :, i:i + 1], f"cross, token {i}")
