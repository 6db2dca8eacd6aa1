"""CPU tier of cross attention and relative position bias: the oracle against
independent forms, the buckets, and the refusals of the C ABI and the Python API
(calls that never reach a GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import cuda_amd._lib as L
import cuda_amd.api as api
import cuda_llm
import oracle

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)


def _torch_forward(q, k, v, lens, scale, table, max_distance, causal):
    """The written-out formula, in torch (autograd)."""
    b, hq, sq, _ = q.shape
    skv = k.shape[2]
    g = hq // k.shape[1]
    x = q @ k.repeat_interleave(g, 1).transpose(2, 3) * scale
    if table is not None:
        ids = torch.tensor([[oracle.relative_bucket(j - i, table.shape[0], causal, max_distance)
                             for j in range(skv)] for i in range(sq)])
        x = x + table[ids].permute(2, 0, 1)
    keep = torch.arange(skv)[None, :] < torch.tensor(lens)[:, None]
    keep = keep[:, None, None, :].expand(b, 1, sq, skv)
    if causal:
        keep = keep & torch.ones(sq, skv, dtype=torch.bool).tril()
    x = x.masked_fill(~keep, -math.inf)
    return torch.softmax(x, -1) @ v.repeat_interleave(g, 1)


@pytest.mark.parametrize("buckets,causal,sq,skv,lens", [
    (0, False, 5, 9, [9, 4]), (8, False, 9, 9, [9, 6]), (6, True, 9, 9, [9, 5]), (8, False, 4, 11, [1, 11])])
def test_oracle_against_autograd_and_differences(buckets, causal, sq, skv, lens):
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(2, h, s, 8, dtype=torch.float64, generator=g)
                   for h, s in ((4, sq), (2, skv), (2, skv), (4, sq)))
    table = torch.randn(buckets, 4, dtype=torch.float64, generator=g) if buckets else None
    leaves = [t.requires_grad_() for t in (q, k, v, table) if t is not None]
    out = _torch_forward(q, k, v, lens, 0.3, table, 12, causal)
    ref = torch.autograd.grad(out, leaves, do)
    n = [t.detach().numpy() if t is not None else None for t in (q, k, v, table)]
    fwd = oracle.encdec_attention(*n[:3], lens, 0.3, n[3], 12, causal)
    np.testing.assert_allclose(fwd["out"], out.detach().numpy(), atol=1e-12)
    got = oracle.encdec_backward(*n[:3], do.numpy(), fwd, lens, 0.3, buckets)
    for name, r in zip(("dq", "dk", "dv", "dtable"), ref):
        np.testing.assert_allclose(got[name], r.numpy(), atol=1e-12)
    # differences along a random direction of every input
    rng = np.random.default_rng(0)
    for i, name in enumerate(("dq", "dk", "dv", "dtable")[:len(leaves)]):
        step = rng.standard_normal(n[i].shape)
        f = []
        for h in (1e-5, -1e-5):
            m = list(n)
            m[i] = n[i] + h * step
            f.append((oracle.encdec_attention(*m[:3], lens, 0.3, m[3], 12, causal)["out"] * do.numpy()).sum())
        assert abs((f[0] - f[1]) / 2e-5 - (got[name] * step).sum()) < 1e-7


def test_oracle_is_plain_attention_at_equal_lengths():
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((2, 2, 7, 8)) for _ in range(3))
    ref = oracle.attention(q, k, v, is_causal=True, scale=0.4, dtype=np.float64)
    flat = np.full((4, 2), 1.5)   # the same bias everywhere: none at all
    got = oracle.encdec_attention(q, k, v, [7, 7], 0.4, flat, 9, True)
    np.testing.assert_allclose(got["out"], ref, atol=1e-12)
    # one query at the end of its keys is the last row of a causal call
    for n in (1, 5, 7):
        table = rng.standard_normal((6, 2))
        whole = oracle.encdec_attention(q, k, v, [n, n], 0.4, table, 5, True)
        one = oracle.encdec_attention(q[:, :, n - 1:n], k, v, [n, n], 0.4, table, 5, True, at_end=True)
        np.testing.assert_allclose(one["out"][:, :, 0], whole["out"][:, :, n - 1], atol=1e-12)


@pytest.mark.parametrize("buckets,causal,distance", [
    (32, False, 128), (32, True, 128), (64, True, 500), (256, True, 2048), (10, False, 20), (4, False, 2),
    (2, True, 2), (8, False, 2048), (12, True, 7), (256, False, 65), (3, True, 2)])
def test_bucket_starts(buckets, causal, distance):
    starts = list(api._bucket_starts(buckets, causal, distance)[0])
    side = buckets if causal else buckets // 2
    e, span = side // 2, side - side // 2
    assert len(starts) == side and starts[0] == 0 and starts == sorted(starts) and starts[-1] <= distance
    last = 0
    for n in range(0, 3 * distance):
        b = max(i for i in range(side) if starts[i] <= n)
        assert b == oracle.relative_bucket(-n, buckets, causal, distance)
        assert b >= last
        last = b
        if not causal and n:
            assert oracle.relative_bucket(n, buckets, causal, distance) == b + side
        x = math.log(max(n, 1) / e) / math.log(distance / e) * span if n >= e else None
        if x is not None and abs(x - round(x)) > 1e-6:   # away from the borders: the closed form
            assert b == min(e + int(x), side - 1)
    # borders that are whole numbers are reached, not missed by a rounding
    if (buckets, causal, distance) == (32, False, 128):
        assert [starts[i] for i in (8, 10, 12, 14)] == [8, 16, 32, 64]
    if causal:
        assert all(oracle.relative_bucket(n, buckets, True, distance) == 0 for n in range(5))


@pytest.mark.parametrize("buckets,causal,distance", [
    (64, True, 20), (64, True, 32), (64, True, 33), (32, False, 8), (32, False, 1), (256, True, 128), (2, True, 1)])
def test_bucket_starts_of_short_distances(buckets, causal, distance):
    """A max_distance that the one-distance buckets pass: from their end on all
    distances are in the last bucket (33: the powers are within one whole number)."""
    starts = list(api._bucket_starts(buckets, causal, distance)[0])
    side = buckets if causal else buckets // 2
    e = side // 2
    assert starts == list(range(e)) + [e] + [max(e, distance)] * (side - e - 1)
    for n in range(3 * side):
        assert oracle.relative_bucket(-n, buckets, causal, distance) == max(i for i in range(side) if starts[i] <= n)
        if n >= max(e, distance):
            assert oracle.relative_bucket(-n, buckets, causal, distance) == side - 1


def test_wrong_buckets_are_noticed():
    """A border one off moves weights by far more than the GPU tests allow."""
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((1, 1, 40, 64)) for _ in range(3))
    t = 2 * rng.standard_normal((8, 1))
    a = oracle.encdec_attention(q, k, v, [40], 0.125, t, 20)["out"]
    b = oracle.encdec_attention(q, k, v, [40], 0.125, t, 30)["out"]   # the side's last bucket from 8, not 7
    assert np.abs(a - b).max() > 2.0 ** -4


SIZES = (2, 4, 2, 8, 9, 64)


def _cross(dtype=L.CA_BF16, q=P, k=P, v=P, lens=None, o=P, lse=None, sizes=SIZES, scale=0.1, ws=P, nbytes=1 << 30):
    return L.load().ca_cross_attention(dtype, q, k, v, lens, o, lse, *sizes, scale, ws, nbytes, None)


def _starts(*x):
    return (ctypes.c_int32 * len(x))(*x)


GOOD = _starts(0, 1, 2, 5)


def _bias(table=P, starts=GOOD, buckets=8, causal=0, sizes=SIZES, scale=0.1, dtype=L.CA_BF16, q=P,
          table_dtype=L.CA_F32, low=None):
    return L.load().ca_relative_bias_attention(dtype, q, P, P, table, table_dtype, starts, buckets, None, P, low, None, *sizes, scale,
                                               causal, P, 1 << 30, None)


def _message():
    return L.load().ca_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"), (dict(sizes=(2, 4, 3, 8, 9, 64)), "multiple"), (dict(sizes=(2, 4, 2, 8, 9, 96)), "head_dim"),
    (dict(sizes=(2, 0, 2, 8, 9, 64)), "positive"), (dict(sizes=(-1, 4, 2, 8, 9, 64)), "negative"),
    (dict(sizes=(2, 4, 2, -8, 9, 64)), "negative"), (dict(sizes=(2, 4, 2, 8, -9, 64)), "negative"),
    (dict(scale=math.nan), "finite"), (dict(scale=math.inf), "finite"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(o=None), "null"), (dict(v=ODD), "aligned"), (dict(o=ODD), "aligned"),
    (dict(sizes=(1 << 30, 4, 2, 1 << 20, 9, 64)), "large"), (dict(sizes=(1, 4, 2, 8, (1 << 31) - 1, 64)), "too long"),
    (dict(sizes=(1 << 20, 4096, 4096, 1, 1, 64)), "heads"), (dict(sizes=(2, 4, 2, 1, 9000, 64), nbytes=0), "workspace"),
])
def test_cross_refusals(kw, word):
    assert _cross(**kw) == L.CA_INVALID_ARGUMENT
    assert word in _message()


@pytest.mark.parametrize("kw,word", [
    (dict(buckets=0), "num_buckets"), (dict(buckets=257, causal=1), "num_buckets"), (dict(buckets=7), "num_buckets"),
    (dict(table=None), "null"), (dict(starts=None), "null"), (dict(starts=_starts(1, 2, 3, 4)), "begin"),
    (dict(starts=_starts(0, 3, 2, 4)), "fall"), (dict(starts=_starts(0, 1, 2, 2049)), "2048"),
    (dict(starts=_starts(0, -1, 2, 3)), "fall"), (dict(scale=math.nan), "finite"), (dict(dtype=9), "dtype"),
    (dict(q=ODD), "aligned"), (dict(table_dtype=5), "dtype"),
    (dict(dtype=L.CA_F32, low=P), "16-bit"), (dict(low=ODD), "aligned"),
])
def test_bias_refusals(kw, word):
    assert _bias(**kw) == L.CA_INVALID_ARGUMENT
    assert word in _message()


def test_empty_calls_do_nothing():
    assert _cross(sizes=(0, 4, 2, 8, 9, 64), q=None, k=None, v=None, o=None) == L.CA_OK
    assert _cross(sizes=(2, 4, 2, 0, 9, 64), q=None, k=None, v=None, o=None) == L.CA_OK
    assert _bias(sizes=(0, 4, 2, 8, 9, 64)) == L.CA_OK
    lib = L.load()
    assert lib.ca_relative_bias_decode(L.CA_F16, None, None, None, P, L.CA_F16, GOOD, 4, None, None, 0, 4, 2, 9, 64, 0.1, None,
                                       0, None) == L.CA_OK


def test_backward_refusals():
    lib = L.load()

    def bwd(lse=P, dq=P, ws=P, nbytes=1 << 30, scale=0.1, dtable=P, bias=True):
        if bias:
            return lib.ca_relative_bias_attention_bwd(L.CA_BF16, P, P, P, P, L.CA_F32, GOOD, 8, None, P, None, P, lse, dq, P, P,
                                                      dtable, *SIZES, scale, 0, ws, nbytes, None)
        return lib.ca_cross_attention_bwd(L.CA_BF16, P, P, P, None, P, P, lse, dq, P, P, *SIZES, scale, ws, nbytes,
                                          None)

    for bias in (False, True):
        for kw, word in ((dict(lse=None), "null"), (dict(dq=None), "null"), (dict(dq=ODD), "aligned"),
                         (dict(scale=math.inf), "finite"), (dict(nbytes=8), "workspace"), (dict(ws=None), "workspace"),
                         (dict(ws=ODD), "aligned")):
            assert bwd(bias=bias, **kw) == L.CA_INVALID_ARGUMENT
            assert word in _message()
    assert bwd(dtable=None) == L.CA_INVALID_ARGUMENT
    # the row pairs, and the tiles' parts of the table's gradient
    assert lib.ca_encoder_decoder_bwd_workspace_bytes(2, 4, 300, 0) == 2 * 4 * 300 * 8
    assert lib.ca_encoder_decoder_bwd_workspace_bytes(2, 4, 300, 32) >= 2 * 4 * (300 * 8 + 10 * 32 * 4)
    big = 2 ** 31 - 1
    for bad in ((0, 4, 300, 0), (2, 0, 300, 0), (2, 4, 0, 0), (2, 4, 300, 257), (2, 4, 300, -1), (big, big, big, 1)):
        assert lib.ca_encoder_decoder_bwd_workspace_bytes(*bad) == 0
    assert lib.ca_cross_attention_workspace_bytes(L.CA_BF16, big, big, 1, big, big, 64, 0) == 0
    # the step's: what its call asks at least, or more
    for dt in (L.CA_F32, L.CA_F16, L.CA_BF16):
        for n, hq, hkv, s, d in ((1, 32, 8, 3000, 128), (64, 32, 8, 8192, 64), (3, 5, 1, 1, 64), (1, 1, 1, 1 << 22, 64)):
            least = lib.ca_decode_workspace_bytes(n, hq, d, s)
            assert lib.ca_relative_bias_decode_workspace_bytes(dt, n, hq, hkv, s, d) >= least
    for bad in ((0, 4, 2, 9, 64), (1, 4, 3, 9, 64), (1, 4, 2, 9, 96), (1, 4, 2, -9, 64), (big, big, 1, 9, 64)):
        assert lib.ca_relative_bias_decode_workspace_bytes(L.CA_F32, *bad) == 0
    # lengths that the calls refuse, the other sizes small
    for q_len, kv_len in ((big, 1), (1, big), (1 << 23, 1)):
        assert lib.ca_cross_attention_workspace_bytes(L.CA_BF16, 1, 1, 1, q_len, kv_len, 64, 1) == 0
        assert lib.ca_relative_bias_attention_workspace_bytes(L.CA_BF16, 1, 1, 1, q_len, kv_len, 64, 0) == 0
        assert _cross(sizes=(1, 1, 1, q_len, kv_len, 64)) == L.CA_INVALID_ARGUMENT


def test_python_refusals():
    q = torch.zeros(1, 4, 3, 64)
    k = torch.zeros(1, 2, 5, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_llm.cross_attention(q, k, k)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_llm.relative_bias_attention(q, k, k, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_llm.relative_bias_decode(q[:, :, :1].contiguous(), k, k, torch.zeros(8, 4))
    for buckets, causal, distance in ((1, True, 8), (2, False, 8), (7, False, 8), (258, True, 300), (32, False, 0),
                                      (32, False, 2049), (32, True, -3)):
        with pytest.raises(RuntimeError, match="buckets|max_distance"):
            api._bucket_starts(buckets, causal, distance)
