"""Attention in 64 bits from its definition, with a bound on what 32-bit arithmetic and the operators' roundings may add to each
value.  Test infrastructure; no code of the package."""
import math

import torch


def buckets(rel, count, most, two_sided):
    """Bucket of each distance key - position, borders in whole numbers."""
    side = count // 2 if two_sided else count
    e = side // 2
    n = side - e
    out = torch.empty_like(rel)
    cache = {}
    for r in torch.unique(rel).tolist():
        d = abs(r) if two_sided else max(-r, 0)
        b = d
        if d >= e:
            b = e
            while b < side - 1 and min(d, most) ** n * e ** (b + 1 - e) >= most ** (b + 1 - e) * e ** n:
                b += 1
        cache[r] = b + (side if two_sided and r > 0 else 0)
        out[rel == r] = cache[r]
    return out


def reference(q, k, v, dout=None, *, key_mask=None, key_lens=None, q_start=None, causal=False, scale=None, table=None,
              max_distance=128, bidirectional=True):
    """Returns {name: (value, bound)} in float64 on the CPU; bound is elementwise."""
    dt = q.dtype
    u = 2.0 ** -24                                             # half a step of float32
    ub = torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0   # half a step of what is rounded besides the results
    uo = torch.finfo(dt).eps / 2
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    B, H, Tq, D = q.shape
    G, Tk = k.shape[1:3]
    R = H // G
    scale = 1 / math.sqrt(D) if scale is None else scale
    j = torch.arange(Tk)
    start = torch.full((B,), Tk - Tq) if q_start is None else q_start.cpu().long()
    pos = torch.arange(Tq)[None] + start[:, None]              # [B, Tq]
    ok = torch.ones(B, Tq, Tk, dtype=torch.bool)
    if key_lens is not None:
        ok &= (j[None] < key_lens.cpu()[:, None])[:, None]
    if key_mask is not None:
        ok &= ~key_mask.cpu()[:, None]
    if causal:
        ok &= j[None, None] <= pos[:, :, None]
    used = ok.any(1)                                           # keys that some query of the row may use
    clean = used[:, None, :, None]
    k, v = torch.where(clean, k, 0.0), torch.where(clean, v, 0.0)
    ke, ve = k.repeat_interleave(R, 1), v.repeat_interleave(R, 1)
    s = (q @ ke.transpose(-1, -2)) * scale
    a = (q.abs() @ ke.abs().transpose(-1, -2)) * abs(scale)
    which = None
    if table is not None:
        which = buckets(j[None, None] - pos[:, :, None], table.shape[0], max_distance, bidirectional)
        t = table.detach().double().cpu()
        bias = t[which].permute(0, 3, 1, 2)
        s = s + bias
        a = a + torch.where(torch.isfinite(bias), bias.abs(), 0.0)
    s = torch.where(ok[:, None], s, -math.inf)
    top = s.amax(-1, keepdim=True) if Tk else torch.full((B, H, Tq, 1), -math.inf, dtype=torch.float64)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(s - top)
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
    lse = torch.where(l > 0, torch.log(torch.where(l > 0, l, 1.0)) + top, -math.inf)[..., 0]
    # a score: D products and sums, scaling, the bias, the change to log2 units; its exponential's relative error is twice that
    # (its own and its row's maximum or log-sum-exp); three roundings of the exponential, the sum and the quotient
    reach = torch.where(ok[:, None], a, 0.0).amax(-1, keepdim=True) if Tk else torch.zeros(B, H, Tq, 1, dtype=torch.float64)
    ds_rel = 2 * (D + 8) * u * reach + (8 + Tk) * u
    out = p @ ve
    pav = p @ ve.abs()
    res = {"out": (out, (ds_rel + ub + (Tk + 4) * u) * pav + uo * out.abs()), "lse": (lse, (ds_rel * 1.0)[..., 0] + 4 * u * torch.nan_to_num(lse.abs(), posinf=0.0))}
    if dout is None:
        return res
    go = dout.detach().double().cpu()
    dv = (p.transpose(-1, -2) @ go).unflatten(1, (G, R)).sum(2)
    dva = ((p * (ds_rel + ub + (Tq * R + 4) * u)).transpose(-1, -2) @ go.abs()).unflatten(1, (G, R)).sum(2)
    dp, dpa = go @ ve.transpose(-1, -2), go.abs() @ ve.abs().transpose(-1, -2)
    delta, da = (go * out).sum(-1, keepdim=True), (go.abs() * pav).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # relative errors of P, of dP (D sums), of delta (the stored, rounded output: uo, ub and its own sums), and dS rounded where it
    # enters a product
    dsa = p * ((ds_rel + ub + (D + 4) * u) * (dpa + da) + (uo + ub + ds_rel + (Tk + D) * u) * da)
    dq, dqa = ds @ ke * scale, (dsa + Tk * u * ds.abs()) @ ke.abs() * abs(scale)
    dk = (ds.transpose(-1, -2) @ q).unflatten(1, (G, R)).sum(2) * scale
    dka = ((dsa + Tq * R * u * ds.abs()).transpose(-1, -2) @ q.abs()).unflatten(1, (G, R)).sum(2) * abs(scale)
    tiny = 1e-30
    res |= {"dq": (dq, dqa + uo * dq.abs() + tiny), "dk": (dk, dka + uo * dk.abs() + tiny), "dv": (dv, dva + uo * dv.abs() + tiny)}
    if table is not None:
        n = table.shape[0]
        hot = torch.nn.functional.one_hot(which, n).double().flatten(0, 2)      # [B Tq Tk, n]
        flat = ds.permute(0, 2, 3, 1).flatten(0, 2)
        # here delta is a 32-bit sum over the keys (bfloat16) or comes from a 32-bit output (float32)
        dta = (p * ((2 * ds_rel + (Tk + 2 * D + 8) * u) * (dpa + da))).permute(0, 2, 3, 1).flatten(0, 2)
        res["dtable"] = (hot.t() @ flat, hot.t() @ dta + (64 + Tq) * u * (hot.t() @ flat.abs()) + tiny)
    return res


def check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = torch.isinf(value) & (got == value)
    off = torch.where(same, 0.0, (got - value).abs())
    bad = ~(off <= bound)
    if bad.any():
        at = tuple(int(x[0]) for x in torch.nonzero(bad, as_tuple=True))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {float(got[at])}, want {float(value[at])} +- {float(bound[at])}; "
                             f"largest difference {float(torch.nan_to_num(off, nan=math.inf).max())}")
