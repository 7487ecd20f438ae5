"""Cases for the self-attention operators: attention forward, attention with its backward pass, and the relative position
bias with its gradient.

``listed()`` gives fixed cases, ``draw()`` more of the same ranges, ``prepare()`` makes a case's inputs, ``run()`` makes one
pass and ``exact()`` says in 64 bits what that pass returns.  ``run()`` computes in plain torch operations while ``own`` is
false and calls wavernn_amd's operators where it is true."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _attention(name, op, dtype, batch, heads, q_len, k_len, dim, *, kv_heads=0, causal=False, padding="none", packed=False,
               buckets=0, distance=128, two_sided=True, cache=False):
    return dict(name=name, op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads or heads, q_len=q_len, k_len=k_len,
                dim=dim, causal=causal, padding=padding, packed=packed, buckets=buckets, distance=distance,
                two_sided=two_sided, cache=cache)


def _bias(name, op, dtype, heads, q_len, k_len, buckets, distance, two_sided):
    return dict(name=name, op=op, dtype=dtype, heads=heads, q_len=q_len, k_len=k_len, buckets=buckets, distance=distance,
                two_sided=two_sided)


def listed():
    return [
        # one utterance through a block of FastPitch's token transformer (generate): latency
        _attention("utterance", "forward", "float32", 1, 2, 128, 128, 128, packed=True),
        # a padded batch through a block of the frame transformer: 640 frames as in the decoder benchmark, ragged lengths
        _attention("frames padded", "forward", "float32", 32, 2, 640, 640, 128, padding="mask", packed=True),
        # one new token of eight streams against long caches of different fill, grouped heads
        _attention("one token, long cache", "forward", "bfloat16", 8, 16, 1, 8191, 128, kv_heads=4, padding="lens", cache=True),
        # a batch of long frame sequences with the learned position bias, in bfloat16
        _attention("frames with bias", "forward", "bfloat16", 4, 8, 1250, 1250, 64, padding="mask", buckets=32),
        # a long causal prompt, grouped heads: the largest forward pass
        _attention("long causal", "forward", "bfloat16", 2, 16, 8192, 8192, 128, kv_heads=4, causal=True),
        # training step of a duration / pitch / energy predictor: short padded token sequences
        _attention("predictor step", "train", "float32", 32, 2, 150, 150, 64, padding="mask", packed=True),
        # training step of the frame transformer with the position bias
        _attention("frames step with bias", "train", "float32", 16, 2, 640, 640, 128, padding="mask", packed=True, buckets=32),
        # training on long causal sequences, grouped heads
        _attention("causal step", "train", "bfloat16", 4, 16, 2048, 2048, 64, kv_heads=4, causal=True),
        # odd sizes: other numbers of queries and keys, a head dimension between the usual ones, ragged lengths, bias
        _attention("odd step", "train", "bfloat16", 3, 6, 517, 1031, 80, kv_heads=3, padding="lens", buckets=32),
        # the largest training step
        _attention("long causal step", "train", "bfloat16", 1, 16, 8192, 8192, 128, causal=True),
        # the dense bias of one utterance, as an additive mask takes it
        _bias("bias of an utterance", "bias", "float32", 2, 128, 128, 32, 128, True),
        # the dense bias of a long sequence and its gradient
        _bias("bias step", "bias step", "float32", 16, 2048, 2048, 32, 128, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


MOST_PAIRS, MOST_FLOPS = 1 << 30, 14 * (1 << 29) * 128   # scores held in the plain form; the largest listed step


def draw(rng):
    kind = rng.choice(["forward", "forward", "train", "train", "bias"])
    if kind == "bias":
        buckets = rng.choice([16, 32, 64])
        return {k: v for k, v in _bias("", rng.choice(["bias", "bias step"]), rng.choice(list(DTYPES)), rng.choice([1, 2, 4, 6, 16]),
                                       _log(rng, 32, 2048), _log(rng, 32, 2048), buckets, rng.choice([64, 128, 200]),
                                       rng.random() < 0.6).items() if k != "name"}
    while True:
        kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        dim = rng.choice([8, 12, 16, 36, 64, 64, 80, 100, 128, 128, 196, 256])
        batch = _log(rng, 1, 32)
        causal = rng.random() < 0.4
        k_len = _log(rng, 16, 8192)
        cache = kind == "forward" and rng.random() < 0.3
        q_len = rng.choice([1, 1, 2, 5, 16]) if cache else k_len if rng.random() < 0.6 else _log(rng, 16, 8192)
        if (causal or cache) and q_len > k_len:
            q_len = k_len
        pairs = batch * kv_heads * group * q_len * k_len
        if pairs <= MOST_PAIRS and pairs * dim * (4 if kind == "forward" else 14) * (0.5 if causal else 1) <= MOST_FLOPS \
                and batch * kv_heads * k_len * dim <= 1 << 28:
            break
    buckets = 0 if rng.random() < 0.5 else rng.choice([16, 32, 64])
    packed = not cache and group == 1 and q_len == k_len and rng.random() < 0.5
    return {k: v for k, v in _attention("", kind, rng.choice(list(DTYPES)), batch, kv_heads * group, q_len, k_len, dim, kv_heads=kv_heads,
                                        causal=causal and not cache, padding="lens" if cache else rng.choice(["none", "mask", "lens"]),
                                        packed=packed, buckets=buckets, distance=rng.choice([64, 128, 200]),
                                        two_sided=not (causal or cache), cache=cache).items() if k != "name"}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(spread).to(dtype)

    s = dict(case)
    if case["op"].startswith("bias"):
        s["table"] = normal(case["buckets"], case["heads"]).requires_grad_(case["op"] == "bias step")
        if case["op"] == "bias step":
            s["dbias"] = normal(case["heads"], case["q_len"], case["k_len"])
        return s
    B, H, G, Tq, Tk, D = (case[k] for k in ("batch", "heads", "kv_heads", "q_len", "k_len", "dim"))
    train = case["op"] == "train"
    if case["packed"]:    # the views that a packed projection of [time, batch, 3 * heads * dim] gives
        q, k, v = normal(Tq, B, 3, H, D, spread=1.2).permute(2, 1, 3, 0, 4).unbind(0)
    else:
        q, k, v = normal(B, H, Tq, D, spread=1.5), normal(B, G, Tk, D), normal(B, G, Tk, D)
    s["q"], s["k"], s["v"] = (x.detach().requires_grad_(train) for x in (q, k, v))
    lens = torch.randint((Tk + 1) // 2, Tk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    s["key_lens"] = lens if case["padding"] == "lens" else None
    s["key_mask"] = torch.arange(Tk, device="cuda")[None, :] >= lens[:, None] if case["padding"] == "mask" else None
    # a cache: the queries are the last tokens of what each row holds
    s["q_start"] = (lens - Tq).clamp_(min=0) if case["cache"] else None
    s["table"] = torch.randn(case["buckets"], H, generator=g, device="cuda").requires_grad_(train) if case["buckets"] else None
    if train:
        s["dout"] = normal(B, H, Tq, D)
    return s


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    H, Tq, Tk = case["heads"], case["q_len"], case["k_len"]
    if case["op"].startswith("bias"):
        n = H * Tq * Tk
        return {"bytes": n * e * (2 if case["op"] == "bias step" else 1), "flops": n if case["op"] == "bias step" else 0}
    B, G, D = case["batch"], case["kv_heads"], case["dim"]
    fill = 1.0 if case["padding"] == "none" else 0.75    # lengths are spread over the upper half
    low = Tq * (Tk - (Tq - 1) / 2) if Tq <= Tk else Tk * (Tk + 1) / 2
    pairs = B * H * (min(low, Tq * Tk * fill) if case["causal"] else Tq * Tk * fill)
    q, kv = B * H * Tq * D * e, B * G * Tk * D * e * fill
    if case["op"] == "forward":
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * pairs}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * D * pairs}


# ------------------------------------------------------------------ the plain form


def _buckets(distance, count, most, two_sided):
    """Bucket of each key position minus query position."""
    if two_sided:
        count //= 2
        first, d = (distance > 0).long() * count, distance.abs()
    else:
        first, d = 0, (-distance).clamp(min=0)
    exact_ones = count // 2
    far = (d.clamp(min=1).double() / exact_ones).log() / math.log(most / exact_ones) * (count - exact_ones)
    far = exact_ones + (far + 1e-9).floor().long()      # a border lies on a whole number or well off it
    return first + torch.where(d < exact_ones, d, far.clamp(max=count - 1))


def _by_distance(x):
    """[..., Tq, Tk] -> [..., Tq + Tk - 1], in 64 bits: sums over the diagonals, the lowest j - i first."""
    Tq, Tk = x.shape[-2:]
    flat = torch.nn.functional.pad(x.flip(-2).double(), (0, Tq)).flatten(-2)
    return flat[..., :Tq * (Tq + Tk - 1)].unflatten(-1, (Tq, Tq + Tk - 1)).sum(-2)


def _bias_run(s):
    table, Tq, Tk = s["table"].detach(), s["q_len"], s["k_len"]
    at = torch.arange(Tk, device="cuda")[None, :] - (torch.arange(Tq, device="cuda")[:, None] + Tk - Tq)
    bias = table[_buckets(at, s["buckets"], s["distance"], s["two_sided"])].permute(2, 0, 1).contiguous()
    if s["op"] == "bias":
        return bias
    d = _by_distance(s["dbias"])
    which = _buckets(torch.arange(Tq + Tk - 1, device="cuda") - (Tk - 1), s["buckets"], s["distance"], s["two_sided"])
    dtable = torch.zeros(s["buckets"], s["heads"], dtype=torch.float64, device="cuda").index_add_(0, which, d.t())
    return bias, dtable.to(table.dtype)


def _attention_run(s):
    q, k, v = (s[n].detach().float() for n in "qkv")
    B, H, Tq, D = q.shape
    G, Tk = k.shape[1:3]
    k, v = (x.repeat_interleave(H // G, 1) for x in (k, v))
    scale = 1 / math.sqrt(D)
    start = s["q_start"].long() if s["q_start"] is not None else torch.full((B,), Tk - Tq, device="cuda")
    at = torch.arange(Tk, device="cuda") - (torch.arange(Tq, device="cuda")[None, :, None] + start[:, None, None])   # [B, Tq, Tk]
    scores = (q @ k.transpose(-1, -2)).mul_(scale)
    if s["table"] is not None:
        table = s["table"].detach()
        which = _buckets(at if s["q_start"] is not None else at[:1], s["buckets"], s["distance"], s["two_sided"])
        scores += table.t()[:, which].transpose(0, 1)
    none = torch.zeros(B, 1, Tk, dtype=torch.bool, device="cuda")
    if s["key_lens"] is not None:
        none = none | (torch.arange(Tk, device="cuda") >= s["key_lens"][:, None])[:, None]
    if s["key_mask"] is not None:
        none = none | s["key_mask"][:, None]
    if s["causal"]:
        none = none | (at > 0)
    scores.masked_fill_(none[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e38)
    p = scores.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = p @ v
    dtype = s["q"].dtype
    if s["op"] == "forward":
        return out.to(dtype)
    dout = s["dout"].float()
    dv = p.transpose(-1, -2) @ dout
    ds = (dout @ v.transpose(-1, -2)).sub_((dout * out).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ k).mul_(scale)
    dk = (ds.transpose(-1, -2) @ q).mul_(scale)
    dk, dv = (x.unflatten(1, (G, H // G)).sum(2) for x in (dk, dv))
    got = [out.to(dtype), dq.to(dtype), dk.to(dtype), dv.to(dtype)]
    if s["table"] is not None:
        which = _buckets(torch.arange(Tq + Tk - 1, device="cuda") - (Tk - 1), s["buckets"], s["distance"], s["two_sided"])
        d = _by_distance(ds.sum(0))
        got.append(torch.zeros(s["buckets"], H, dtype=torch.float64, device="cuda").index_add_(0, which, d.t()).float())
    return got


# ------------------------------------------------------------------ the framework's operators


def _own_run(s):
    from wavernn_amd.attention import attention, relative_position_bias
    bias = dict(max_distance=s["distance"], bidirectional=s["two_sided"])
    if s["op"] == "bias":
        return relative_position_bias(s["table"], s["q_len"], s["k_len"], **bias)
    if s["op"] == "bias step":
        out = relative_position_bias(s["table"], s["q_len"], s["k_len"], **bias)
        return out.detach(), torch.autograd.grad(out, s["table"], s["dbias"])[0]
    out = attention(s["q"], s["k"], s["v"], key_mask=s["key_mask"], key_lens=s["key_lens"], q_start=s["q_start"],
                    causal=s["causal"], bias_table=s["table"], **bias)
    if s["op"] == "forward":
        return out
    leaves = [s["q"], s["k"], s["v"]] + ([s["table"]] if s["table"] is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def run(state):
    if own:
        return _own_run(state)
    return _bias_run(state) if state["op"].startswith("bias") else _attention_run(state)


# ------------------------------------------------------------------ the definition in 64 bits


def _edges(count, most):
    """The distances at which a bucket above the exact ones begins, in whole numbers."""
    e = count // 2
    n = count - e
    found = []
    for k in range(1, n):
        d = e
        while d ** n * e ** k < most ** k * e ** n:
            d += 1
        found.append(d)
    return e, torch.tensor(found, dtype=torch.int64)


def _bucket_map(Tq, Tk, start, count, most, two_sided):
    rel = torch.arange(Tk)[None, :] - torch.arange(Tq)[:, None] - start
    side = count // 2 if two_sided else count
    e, edges = _edges(side, most)
    far = rel.abs() if two_sided else (-rel).clamp(min=0)
    which = torch.where(far < e, far, e + torch.bucketize(far, edges, right=True))
    return (which + (rel > 0) * side if two_sided else which).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("bias"):
        table = s["table"].detach().double().requires_grad_()
        hot = _bucket_map(s["q_len"], s["k_len"], s["k_len"] - s["q_len"], s["buckets"], s["distance"], s["two_sided"])
        bias = table.detach()[hot].permute(2, 0, 1)
        if case["op"] == "bias":
            return bias
        d = s["dbias"].double()
        return bias, torch.stack([d[:, hot == n].sum(-1) for n in range(s["buckets"])])
    q, k, v = (s[n].detach().double() for n in "qkv")
    B, H, Tq, D = q.shape
    G, Tk = k.shape[1:3]
    train = case["op"] == "train"
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros(s["buckets"], H, dtype=torch.float64, device="cuda")
    hot = None
    for b in range(B):
        start = int(s["q_start"][b]) if s["q_start"] is not None else Tk - Tq
        j = torch.arange(Tk, device="cuda")
        ok = torch.ones(Tq, Tk, dtype=torch.bool, device="cuda")
        if s["key_lens"] is not None:
            ok &= j < int(s["key_lens"][b])
        if s["key_mask"] is not None:
            ok &= ~s["key_mask"][b]
        if case["causal"]:
            ok &= j <= torch.arange(Tq, device="cuda")[:, None] + start
        some = ok.any(1, keepdim=True)
        if s["table"] is not None and (hot is None or s["q_start"] is not None):
            hot = _bucket_map(Tq, Tk, start, s["buckets"], s["distance"], s["two_sided"])
        for h in range(H):
            kh, vh = k[b, h // (H // G)], v[b, h // (H // G)]
            x = q[b, h] @ kh.t() / D ** 0.5
            if s["table"] is not None:
                x = x + s["table"].detach().double()[:, h][hot]
            p = torch.where(ok, torch.softmax(torch.where(ok, x, -1e300), -1), 0.0) * some
            out[b, h] = p @ vh
            if train:
                do = s["dout"][b, h].double()
                dv[b, h // (H // G)] += p.t() @ do
                dp = do @ vh.t()
                dx = p * (dp - (p * dp).sum(1, keepdim=True))
                dq[b, h] = dx @ kh / D ** 0.5
                dk[b, h // (H // G)] += dx.t() @ q[b, h] / D ** 0.5
                if s["table"] is not None:
                    for n in range(s["buckets"]):
                        dtable[n, h] += dx[hot == n].sum()
    if not train:
        return out
    return [out, dq, dk, dv] + ([dtable] if s["table"] is not None else [])
