"""The encoder-decoder attention operators as they are measured.

``cross`` is attention to an encoder's states of another length over a padded
batch (``cross_attention``), ``cross_train`` its training step, ``cross_step``
one token of generation against the encoder's states. ``bias`` is
self-attention with a learned relative position bias by buckets
(``relative_bias_attention``), ``bias_train`` its training step with the
table's gradient, ``bias_step`` one token of generation over a cache
(``relative_bias_decode``).

Lengths of a batch are spread evenly over [lo, keys] and dealt to the
sequences in an order that depends on the seed, so a case's work does not.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token for three interactive users against short encoder states:
        # latency
        dict(name="cross_step_few", kind="cross_step", dtype="bf16", batch=3, heads=32, kv_heads=8, rows=1,
             keys=333, lo=90, dim=128),
        # one token of a serving batch against long encoder states, as a speech
        # or document encoder leaves them
        dict(name="cross_step_batch", kind="cross_step", dtype="fp16", batch=64, heads=16, kv_heads=16, rows=1,
             keys=1500, lo=300, dim=64),
        # a decoder's prompt of a few rows against one long document
        dict(name="cross_prompt", kind="cross", dtype="bf16", batch=1, heads=32, kv_heads=8, rows=50, keys=4001,
             lo=4001, dim=128),
        # a padded batch of targets against their sources
        dict(name="cross_batch", kind="cross", dtype="bf16", batch=4, heads=32, kv_heads=32, rows=2048,
             keys=4096, lo=1024, dim=128),
        # a cross attention layer's training step, grouped heads, ragged sources
        dict(name="cross_train", kind="cross_train", dtype="bf16", batch=2, heads=32, kv_heads=8, rows=1000,
             keys=4096, lo=1500, dim=128),
        # the same in float32, as small research models run it
        dict(name="cross_train_f32", kind="cross_train", dtype="fp32", batch=2, heads=8, kv_heads=8, rows=300,
             keys=1024, lo=700, dim=64),
        # a short text through one encoder layer: few tiles, latency
        dict(name="bias_short", kind="bias", dtype="bf16", batch=1, heads=12, kv_heads=12, rows=100, keys=100,
             lo=100, dim=64, causal=False, buckets=32, distance=128),
        # a padded batch of paragraphs through an encoder layer
        dict(name="bias_batch", kind="bias", dtype="fp16", batch=16, heads=16, kv_heads=16, rows=512, keys=512,
             lo=64, dim=64, causal=False, buckets=32, distance=128),
        # a long document, causal
        dict(name="bias_long", kind="bias", dtype="bf16", batch=1, heads=32, kv_heads=32, rows=8192, keys=8192,
             lo=8192, dim=64, causal=True, buckets=32, distance=128),
        # an encoder layer's training step over a padded batch
        dict(name="bias_train", kind="bias_train", dtype="bf16", batch=8, heads=16, kv_heads=16, rows=1024,
             keys=1024, lo=200, dim=64, causal=False, buckets=32, distance=128),
        # a decoder layer's training step, grouped heads, wider buckets
        dict(name="bias_train_causal", kind="bias_train", dtype="fp16", batch=2, heads=32, kv_heads=8, rows=2000,
             keys=2000, lo=2000, dim=128, causal=True, buckets=64, distance=500),
        # one token of a serving batch over a cache
        dict(name="bias_step", kind="bias_step", dtype="bf16", batch=32, heads=32, kv_heads=32, rows=1, keys=4096,
             lo=100, dim=64, causal=True, buckets=32, distance=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, key heads)
_HEADS = [(32, 8), (32, 32), (16, 16), (8, 8), (24, 4), (32, 4), (12, 12)]
# no drawn case does more than about the largest listed one of its kind
_MOST_FLOPS = {"cross": 3.9e11, "cross_train": 3.9e11, "bias": 2.7e11, "bias_train": 2.3e11}
_MOST_BYTES = {"cross_step": 2.4e8, "bias_step": 5.5e8}


def draw(rng):
    kind = rng.choice(["cross_step", "cross", "cross", "cross_train", "bias", "bias", "bias_train", "bias_step"])
    while True:
        heads, kv_heads = rng.choice(_HEADS)
        keys = _log_int(rng, 1 if rng.random() < 0.1 else 30, 8192)
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), heads=heads, kv_heads=kv_heads,
                    keys=keys, dim=rng.choice([64, 128]))
        if kind.endswith("_step"):
            case.update(batch=_log_int(rng, 1, 100), rows=1)
        else:
            case.update(batch=rng.choice([1, 1, 2, 3, 4, 8]), rows=_log_int(rng, 2, 8192))
        if kind.startswith("bias"):
            if kind != "bias_step":
                case["rows"] = keys
            case.update(causal=kind == "bias_step" or rng.random() < 0.5, buckets=rng.choice([32, 32, 64, 10]),
                        distance=rng.choice([128, 128, 20, 500, 1000]))
        # now and then a sequence of the batch has no key at all
        case["lo"] = 0 if rng.random() < 0.1 else max(1, int(keys * rng.choice([0.03, 0.25, 1.0])))
        if not sum(_lens(case)):
            continue
        w = work(case)
        most = _MOST_FLOPS.get(kind, math.inf)
        if case["dtype"] == "fp32":   # float32 products run at about a sixteenth of the rate
            most /= 16
        if w["flops"] <= most and w["bytes"] <= _MOST_BYTES.get(kind, math.inf):
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case, order=None):
    """Key lengths, spread evenly over [lo, keys] (keys itself among them)."""
    n, lo, hi = case["batch"], case["lo"], case["keys"]
    lens = [hi - (hi - lo) * i // n for i in range(n)]
    return lens if order is None else [lens[i] for i in order]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed)).tolist()
    dtype = _DTYPES[case["dtype"]]
    b, hq, hkv, m, n, d = (case[x] for x in ("batch", "heads", "kv_heads", "rows", "keys", "dim"))

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    state = dict(case=case, q=normal(b, hq, m, d), k=normal(b, hkv, n, d), v=normal(b, hkv, n, d),
                 lens=torch.tensor(_lens(case, order), dtype=torch.int32, device="cuda"))
    if case["kind"].startswith("bias"):
        # a trained table's entries differ by a few units between near and far
        state["table"] = normal(case["buckets"], hq) * 2
    if case["kind"].endswith("train"):
        state["dout"] = normal(b, hq, m, d)
        for name in ("q", "k", "v", "table"):
            if name in state:
                state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _own(s):
    import cuda_llm

    case, kind = s["case"], s["case"]["kind"]
    if kind == "bias_step":
        return cuda_llm.relative_bias_decode(s["q"], s["k"], s["v"], s["table"], s["lens"],
                                             max_distance=case["distance"])
    if kind.startswith("bias"):
        out = cuda_llm.relative_bias_attention(s["q"], s["k"], s["v"], s["table"], s["lens"],
                                               is_causal=case["causal"], max_distance=case["distance"])
    else:
        out = cuda_llm.cross_attention(s["q"], s["k"], s["v"], s["lens"])
    if not kind.endswith("train"):
        return out
    names = [x for x in ("q", "k", "v", "table") if x in s]
    grads = torch.autograd.grad(out, [s[x] for x in names], s["dout"])
    return {"out": out.detach(), **{"d" + x: t for x, t in zip(names, grads)}}


def _buckets(case, distance):
    """Bucket of key position - query position, elementwise."""
    side = case["buckets"]
    if case["causal"]:
        n, base = (-distance).clamp_min(0), 0
    else:
        side //= 2
        n, base = distance.abs(), torch.where(distance > 0, side, 0)
    exact_ = side // 2
    far = torch.log(n.clamp_min(1).double() / exact_) / math.log(case["distance"] / exact_) * (side - exact_)
    # (a border that the logarithms reach but for their rounding counts as reached)
    far = (exact_ + torch.floor(far + 1e-9)).clamp_max(side - 1).long()
    return base + torch.where(n < exact_, n, far)


def _plain(s):
    case = s["case"]
    kind, dtype = case["kind"], s["q"].dtype
    q, k, v = (s[x].detach().float() for x in "qkv")
    b, hq, m, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d)
    lens = s["lens"].long()
    cols = torch.arange(n, device=q.device)
    valid = (cols[None, :] < lens[:, None])[:, None, None, :]            # [b, 1, 1, n]
    # what padded rows hold takes no part
    keep = valid.transpose(2, 3)
    k, v = torch.where(keep, k, 0.0), torch.where(keep, v, 0.0)
    group = hq // hkv
    q4 = q.view(b, hkv, group * m, d)
    x = torch.matmul(q4, k.transpose(2, 3).contiguous()).view(b, hq, m, n) * scale
    bucket = None
    if kind.startswith("bias"):
        rows = torch.arange(m, device=q.device)
        if kind == "bias_step":
            distance = cols[None, :] - (lens[:, None] - 1)                # [b, n]
            bucket = _buckets(case, distance)
            x += s["table"].detach().float()[bucket].permute(0, 2, 1)[:, :, None, :]
        else:
            distance = cols[None, :] - rows[:, None]
            bucket = _buckets(case, distance)
            x += s["table"].detach().float().t().contiguous()[:, bucket]
            if case["causal"]:
                valid = valid & (distance <= 0)
    x = torch.where(valid, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    del x
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    p4 = p.view(b, hkv, group * m, n)
    out = torch.matmul(p4, v).view(b, hq, m, d)
    if not kind.endswith("train"):
        return out.to(dtype)
    do = s["dout"].float()
    do4 = do.view(b, hkv, group * m, d)
    dv = torch.matmul(p4.transpose(2, 3).contiguous(), do4)
    ds = torch.matmul(do4, v.transpose(2, 3).contiguous()).view(b, hq, m, n)
    ds = p * (ds - (do * out).sum(-1, keepdim=True))
    ds4 = ds.view(b, hkv, group * m, n)
    res = {"out": out.to(dtype), "dq": (torch.matmul(ds4, k) * scale).view(b, hq, m, d).to(dtype),
           "dk": (torch.matmul(ds4.transpose(2, 3).contiguous(), q4) * scale).to(dtype), "dv": dv.to(dtype)}
    if bucket is not None:
        # A distance's sum first: with the rows turned round and padded to m + n, reading
        # them at m + n - 1 a row puts every distance in a column of its own. (A bucket's
        # is of millions of terms of both signs: 64 bits.)
        skew = torch.zeros(hq, m, m + n, device=q.device)
        skew[:, :, :n] = ds.sum(0).flip(1)
        skew = skew.view(hq, -1)[:, :m * (m + n - 1)].view(hq, m, m + n - 1)
        per = skew.sum(1, dtype=torch.float64)
        dtable = torch.zeros(case["buckets"], hq, dtype=torch.float64, device=q.device)
        at = _buckets(case, torch.arange(1 - m, n, device=q.device))
        dtable.index_add_(0, at, per.t().contiguous())
        res["dtable"] = dtable.to(s["table"].dtype)
    return res


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    elem = 4 if case["dtype"] == "fp32" else 2
    b, hq, hkv, m, d = (case[x] for x in ("batch", "heads", "kv_heads", "rows", "dim"))
    lens = _lens(case)
    if case.get("causal") and case["kind"] != "bias_step":
        pairs = sum(n * (n + 1) // 2 + (m - n) * n if n < m else m * (m + 1) // 2 for n in lens)
    else:
        pairs = m * sum(lens)
    product = 2 * hq * pairs * d
    rows_q, rows_kv = b * hq * m * d, hkv * sum(lens) * d
    table = case["buckets"] * hq * elem if "buckets" in case else 0
    if case["kind"].endswith("train"):
        # q, dout, k, v in; out, dq and all of dk, dv out; two and five products
        total = 4 * rows_q + 2 * rows_kv + 2 * b * hkv * case["keys"] * d
        return {"bytes": total * elem + 2 * table + 4 * b, "flops": 7 * product}
    return {"bytes": (2 * rows_q + 2 * rows_kv) * elem + table + 4 * b, "flops": 2 * product}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------
def _first_distances(side, most):
    """First distance of each bucket of a side, in whole numbers."""
    e = side // 2
    span = side - e
    first = list(range(e))
    n = e
    for j in range(span):
        # n / e >= (most / e) ^ (j / span)
        while n ** span * e ** j < most ** j * e ** span:
            n += 1
        first.append(n)
    return first


def _bias_by_distance(case, table, distances):
    """table rows [len(distances), heads] in 64 bits, and their indices."""
    causal = case["causal"]
    side = case["buckets"] if causal else case["buckets"] // 2
    first = _first_distances(side, case["distance"])
    ids = []
    for x in distances:
        n = max(-x, 0) if causal else abs(x)
        b = max(i for i in range(side) if first[i] <= n)
        ids.append(b + (side if x > 0 and not causal else 0))
    ids = torch.tensor(ids, device=table.device)
    return table.double()[ids], ids


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        q, k, v = (s[x].detach() for x in "qkv")
        b, hq, m, d = q.shape
        ratio, n_all = hq // k.shape[1], k.shape[2]
        scale = d ** -0.5
        f64 = dict(dtype=torch.float64, device=q.device)
        out = torch.zeros(b, hq, m, d, **f64)
        grads = {x: torch.zeros(s[x].shape, **f64) for x in ("q", "k", "v", "table")
                 if x in s and kind.endswith("train")}
        if kind.startswith("bias"):
            # entry i of the vector is distance i - offset
            offset = n_all + m
            rows64, ids = _bias_by_distance(case, s["table"].detach(), range(-offset, offset + 1))
        for i, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            for h in range(hq):
                kk, vv = k[i, h // ratio, :n].double(), v[i, h // ratio, :n].double()
                qq = q[i, h].double()
                logits = scale * (qq @ kk.t())
                if kind.startswith("bias"):
                    at = torch.arange(m, device=q.device) if kind != "bias_step" else torch.tensor(
                        [n - 1], device=q.device)
                    dist = torch.arange(n, device=q.device).view(1, -1) - at.view(-1, 1)
                    logits += rows64[:, h][dist + offset]
                    if case["causal"]:
                        logits.masked_fill_(dist > 0, -math.inf)
                p = torch.softmax(logits, -1)
                out[i, h] = p @ vv
                if grads:
                    do = s["dout"][i, h].double()
                    grads["v"][i, h // ratio, :n] += p.t() @ do
                    ds = p * (do @ vv.t() - (do * out[i, h]).sum(-1, keepdim=True))
                    grads["q"][i, h] = scale * (ds @ kk)
                    grads["k"][i, h // ratio, :n] += scale * (ds.t() @ qq)
                    if "table" in grads:
                        grads["table"][:, h] += torch.bincount(ids[dist + offset].view(-1), ds.reshape(-1),
                                                               minlength=case["buckets"])
    return {"out": out, **{"d" + x: t for x, t in grads.items()}} if grads else out
