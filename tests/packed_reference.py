"""64-bit references of the packed and paged operators, one sequence and one head
at a time, and how far a result may be off.

Bounds, element by element: `u` = half a step of the element type relative to a
value (finfo.eps / 2).  A result is rounded once (u |x|); the probabilities, and
in the backward the score gradients, are rounded once before their products (u of
the sum of magnitudes); fp32 sums, exp and the statistics give `C` of that sum:
scores of D terms are off by at most D 2^-24 sum |q||k| scale (below 1e-5 for the
unit normal rows here: 128 x 6e-8 x 11), exp2 and the row sum by a few 2^-24 more."""
import math

import torch

C = 2e-5


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def packed(q, k, v, bounds, scale, do=None):
    """{name: (value, bound)} of o, lse and, with do, dq, dk, dv (float64)."""
    u, G = half_step(q.dtype), q.shape[1] // k.shape[1]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=q.device)  # noqa: E731
    out = {n: [z(t), z(t)] for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    lse = torch.zeros(q.shape[1], q.shape[0], dtype=torch.float64, device=q.device)
    for a, b in zip(bounds[:-1], bounds[1:]):
        for h in range(q.shape[1] if b > a else 0):
            qh, kh, vh = (t[a:b, i].double() for t, i in ((q, h), (k, h // G), (v, h // G)))
            s = (qh @ kh.T) * scale
            s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
            lse[h, a:b] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[h, a:b, None])
            o = p @ vh
            eo = u * o.abs() + (u + C) * (p @ vh.abs())
            out["o"][0][a:b, h], out["o"][1][a:b, h] = o, eo
            if do is None:
                continue
            dh = do[a:b, h].double()
            dp = dh @ vh.T
            delta = (dh * o).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            # Delta comes from the rounded o; dp and Delta are fp32 sums
            e = (dh.abs() * eo).sum(1, keepdim=True) + C * (dh.abs() @ vh.abs().T + (dh * o).abs().sum(1, keepdim=True))
            es = (u + C) * ds.abs() + p * e * scale
            out["dq"][0][a:b, h] = ds @ kh
            out["dq"][1][a:b, h] = u * (ds @ kh).abs() + es @ kh.abs()
            out["dk"][0][a:b, h // G] += ds.T @ qh
            out["dk"][1][a:b, h // G] += es.T @ qh.abs()
            out["dv"][0][a:b, h // G] += p.T @ dh
            out["dv"][1][a:b, h // G] += (u + C) * (p.T @ dh.abs())
    for n in ("dk", "dv"):
        out[n][1] += u * out[n][0].abs()
    out["lse"] = [lse, C * (1 + lse.abs())]
    return {n: x for n, x in out.items() if do is not None or n in ("o", "lse")}


def near(name, got, want, rows=None):
    """got against (value, bound), with a smallest normal of the type to spare."""
    value, bound = want
    got = got.double()
    tiny = 2.0 ** -24 if name != "lse" else 0.0
    over = ((got - value).abs() - bound - tiny)
    if rows is not None:
        over = over[:rows] if name != "lse" else over[:, :rows]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0.0, f"{name}: {worst:.3e} over its bound (nan: {bool(torch.isnan(over).any())})"
    assert not torch.isnan(over).any(), name


def quantise(x):
    """(codes, scales) of an 8-bit cache."""
    # divided in 64 bits and rounded once (in 32, torch's division by a number is a
    # product with its reciprocal on the GPU, up to a step off)
    scale = (x.double().abs().amax(-1) / 127.0).float().clamp_min(2.0 ** -126)
    codes = (x.double() / scale.double()[..., None]).round().clamp(-127, 127)
    return codes.to(torch.int8), scale


def decode(q, kc, vc, table, lens, scale, ks=None, vs=None):
    """{o: (value, bound), lse: ..}, of a cache [pages][HK][P][D]."""
    u, (B, H, D), P = half_step(q.dtype), q.shape, kc.shape[2]
    G = H // kc.shape[1]
    o = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    eo, lse = torch.zeros_like(o), torch.full((B, H), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        ids = table[b, :-(-n // P)].long()
        kv = []
        for c, s in ((kc, ks), (vc, vs)):
            x = c[ids].double() if s is None else c[ids].double() * s[ids].double()[..., None]
            kv.append(x.transpose(0, 1).reshape(c.shape[1], -1, D)[:, :n])
        for h in range(H):
            x = (kv[0][h // G] @ q[b, h].double()) * scale
            lse[b, h] = torch.logsumexp(x, 0)
            p = torch.exp(x - lse[b, h])
            o[b, h] = p @ kv[1][h // G]
            # (fp16 holds weights below 2^-14 of the largest to 2^-25 of it)
            small = n * 2.0 ** -24 * float(kv[1][h // G].abs().max()) if q.dtype == torch.float16 else 0.0
            eo[b, h] = u * o[b, h].abs() + (u + C) * (p @ kv[1][h // G].abs()) + small
    return {"o": [o, eo], "lse": [lse, C * (1 + lse.abs().nan_to_num(0.0, 0.0, 0.0))]}
