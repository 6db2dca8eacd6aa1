"""fp64 math of the encoder-decoder operators — test infrastructure only.

Cross attention (keys of another length, padded per sequence) and attention
with a learned relative position bias by buckets, with their gradients. No
reference counterpart: the definitions are the docstrings of
``cuda_llm.cross_attention_forward`` and ``relative_bias_attention_forward``.
"""
import numpy as np


def relative_bucket(distance, num_buckets, is_causal, max_distance):
    """Bucket of a key `distance` after its query (an int), by whole numbers."""
    side = num_buckets if is_causal else num_buckets // 2
    n = max(-distance, 0) if is_causal else abs(distance)
    e = side // 2
    span = side - e
    b = n
    if n >= e:
        # the largest j with (n / e) ** span >= (max_distance / e) ** j
        j = 0
        while j + 1 < span and n ** span * e ** (j + 1) >= max_distance ** (j + 1) * e ** span:
            j += 1
        b = e + j
    return b + (side if distance > 0 and not is_causal else 0)


def bucket_matrix(rows, keys, num_buckets, is_causal, max_distance, first_row=0):
    """[rows, keys] bucket ids; query i is at position first_row + i."""
    lo, hi = -(first_row + rows - 1), keys - 1 - first_row
    ids = np.array([relative_bucket(x, num_buckets, is_causal, max_distance) for x in range(lo, hi + 1)], dtype=int)
    d = np.arange(keys)[None, :] - (first_row + np.arange(rows))[:, None]
    return ids[d - lo] if keys else np.zeros((rows, 0), dtype=int)


def encdec_attention(q, k, v, lens, scale, table=None, max_distance=128, is_causal=False, at_end=False):
    """dict(out, lse, p, logits, bucket): q [B, Hq, Sq, D]; k, v [B, Hkv, Skv, D];
    lens [B]; table [buckets, Hq] or None; at_end: each sequence's queries end at
    its last key (decode). p and logits [B, Hq, Sq, Skv] (logits -inf where a key
    takes no part); bucket [B, Sq, Skv] or None."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    b, hq, sq, d = q.shape
    hkv, skv = k.shape[1], k.shape[2]
    lens = np.clip(np.asarray(lens), 0, skv)
    out = np.zeros((b, hq, sq, d))
    lse = np.full((b, hq, sq), -np.inf)
    p = np.zeros((b, hq, sq, skv))
    logits = np.full((b, hq, sq, skv), -np.inf)
    bucket = None if table is None else np.zeros((b, sq, skv), dtype=int)
    for i in range(b):
        n = int(lens[i])
        first = n - sq if at_end else 0
        if table is not None and n:
            bucket[i, :, :n] = bucket_matrix(sq, n, table.shape[0], is_causal, max_distance, first)
        for h in range(hq):
            g = h // (hq // hkv)
            if n == 0 or sq == 0:
                continue
            x = q[i, h] @ k[i, g, :n].T * scale
            if table is not None:
                x = x + np.clip(np.asarray(table, dtype=np.float64), -32768, 32768)[:, h][bucket[i, :, :n]]
                x[np.isneginf(np.asarray(table, dtype=np.float64)[:, h][bucket[i, :, :n]])] = -np.inf
            if is_causal:
                x[np.arange(n)[None, :] > first + np.arange(sq)[:, None]] = -np.inf
            m = x.max(1, keepdims=True)
            e = np.exp(x - np.where(np.isneginf(m), 0, m))
            s = e.sum(1, keepdims=True)
            w = e / np.where(s == 0, 1, s)
            logits[i, h, :, :n], p[i, h, :, :n] = x, w
            out[i, h] = w @ v[i, g, :n]
            lse[i, h] = np.where(s == 0, -np.inf, np.log(np.where(s == 0, 1, s)) + m)[:, 0]
    return dict(out=out, lse=lse, p=p, logits=logits, bucket=bucket)


def encdec_backward(q, k, v, dout, fwd, lens, scale, num_buckets=0, out=None, magnitude=False):
    """dict(dq, dk, dv[, dtable]) from encdec_attention's result; `out`: the output
    that rowsum(dout * out) takes (None: the exact one). magnitude: every product
    and sum of absolute values instead, which bounds what roundings do."""
    q, k, v, dout = (np.asarray(x, dtype=np.float64) for x in (q, k, v, dout))
    o = fwd["out"] if out is None else np.asarray(out, dtype=np.float64)
    if magnitude:
        q, k, v, dout, o = (np.abs(x) for x in (q, k, v, dout, o))
    b, hq, sq, d = q.shape
    hkv, skv = k.shape[1], k.shape[2]
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    dtable = np.zeros((num_buckets, hq))
    for i in range(b):
        n = int(np.clip(lens[i], 0, skv))
        for h in range(hq):
            g = h // (hq // hkv)
            if n == 0:
                continue
            p = fwd["p"][i, h, :, :n]
            row = (dout[i, h] * o[i, h]).sum(1, keepdims=True)
            dp = dout[i, h] @ v[i, g, :n].T
            ds = p * (dp + row if magnitude else dp - row)
            dv[i, g, :n] += p.T @ dout[i, h]
            dq[i, h] = ds @ k[i, g, :n] * abs(scale) if magnitude else ds @ k[i, g, :n] * scale
            dk[i, g, :n] += ds.T @ q[i, h] * (abs(scale) if magnitude else scale)
            if num_buckets:
                np.add.at(dtable[:, h], fwd["bucket"][i, :, :n].ravel(), ds.ravel())
    res = dict(dq=dq, dk=dk, dv=dv)
    if num_buckets:
        res["dtable"] = dtable
    return res
