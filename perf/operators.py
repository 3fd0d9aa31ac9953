"""The operators of serving and training on many sequences at once: packed
prompts with grouped heads, a paged key-value cache, and the attention of one
new token over it.

  prompt   causal attention of packed sequences of different lengths (cu_seqlens),
           each key-value head shared by a group of query heads: o and lse
  train    the same forward, and its backward: o, lse, dq, dk, dv
  cache    a prompt's (or a step's) keys and values into the pages of a cache,
           as they are or in 8 bits with a scale per row, and the rows read
           back: what a request that reuses them attends to
  decode   one query per sequence against the pages its table names, each
           sequence of its own length: o and lse

`own` chooses between the library's entry points and the plain form of the same
calls: elementary torch operations in 32 bits, rounded once at the end.
Sizes are those of the library's own configurations (168-, 384-, 768- and
4096-dim) and ragged ones between them.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


def _wha():
    from __graft_entry__ import load_package
    return load_package()


def listed():
    return [
        # a small model's prompts: the smallest call, where launches and latency count
        dict(name="prompt_168", kind="prompt", S=4, L=256, H=4, HK=2, D=42, dtype="f32", fused=False, empty=False),
        # a serving batch of the production size: ragged prompts, three query heads to a key-value head,
        # q, k and v as they lie in one fused projection's rows
        dict(name="prompt_768", kind="prompt", S=16, L=1024, H=12, HK=4, D=64, dtype="bf16", fused=True, empty=False),
        # long prompts at the widest preset
        dict(name="prompt_4096", kind="prompt", S=4, L=4096, H=32, HK=8, D=128, dtype="bf16", fused=True, empty=False),
        # fine-tuning on packed documents in full precision, a key-value head for each query head
        dict(name="train_384", kind="train", S=16, L=512, H=8, HK=8, D=48, dtype="f32", fused=True, empty=False),
        # the production size in half precision
        dict(name="train_768", kind="train", S=12, L=1024, H=12, HK=4, D=64, dtype="bf16", fused=True, empty=False),
        # long documents at the widest preset: the largest work
        dict(name="train_4096", kind="train", S=4, L=4096, H=32, HK=8, D=128, dtype="bf16", fused=True, empty=False),
        # one step of 64 sequences into an 8-bit cache
        dict(name="cache_step", kind="cache", N=64, HK=12, D=64, dtype="bf16", cache="i8", P=16, pages=4096, fused=True),
        # long prompts into an 8-bit cache, an odd number of rows
        dict(name="cache_prompt_i8", kind="cache", N=16301, HK=8, D=128, dtype="bf16", cache="i8", P=64, pages=512,
             fused=True),
        # a full-precision model's prompts into a cache of its own type
        dict(name="cache_prompt_f32", kind="cache", N=8192, HK=12, D=64, dtype="f32", cache="f32", P=32, pages=512,
             fused=False),
        # a few short conversations, one idle place in the batch: latency counts
        dict(name="decode_768", kind="decode", S=8, L=1024, H=12, HK=4, D=64, dtype="bf16", cache="bf16", P=16,
             empty=True),
        # a full serving batch over an 8-bit cache
        dict(name="decode_4096_i8", kind="decode", S=32, L=8192, H=32, HK=8, D=128, dtype="bf16", cache="i8", P=64,
             empty=False),
        # one very long conversation: few rows, work only along the cache
        dict(name="decode_long", kind="decode", S=1, L=131072, H=32, HK=8, D=128, dtype="bf16", cache="bf16", P=64,
             empty=False),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


_HEAD_DIMS = (32, 40, 42, 48, 56, 64, 64, 80, 96, 100, 128, 128)


def draw(rng):
    """One more case of the listed kinds: sizes spread over their logarithm."""
    kind = rng.choice(("prompt", "prompt", "train", "train", "cache", "decode", "decode"))
    while True:
        HK = rng.choice((1, 2, 4, 4, 8, 8, 12))
        c = dict(kind=kind, HK=HK, D=rng.choice(_HEAD_DIMS))
        if kind == "cache":
            dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
            P = rng.choice((8, 16, 32, 64, 128, 256))
            N = _loguniform(rng, 1, 16301)
            c.update(N=N, dtype=dtype, cache=rng.choice((dtype, "i8", "i8")), P=P,
                     pages=-(-N // P) + rng.randrange(1, 64), fused=rng.random() < 0.5)
            if N * HK * c["D"] * _SIZE[dtype] <= 16301 * 8 * 128 * 2:
                return c
            continue
        c.update(H=HK * rng.choice((1, 1, 2, 3, 4, 8)), empty=rng.random() < 0.25)
        if kind == "decode":
            dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
            c.update(S=_loguniform(rng, 1, 64), L=_loguniform(rng, 1, 131072), dtype=dtype,
                     cache=rng.choice((dtype, "i8")), P=rng.choice((8, 16, 32, 64, 128, 256)))
            rows = c["S"] * c["L"] * HK * c["D"]
            if c["H"] <= 64 and rows * _SIZE[c["cache"]] <= 131072 * 8 * 128 * 2:
                return c
            continue
        # (a gradient in 16-bit floating point would need a scaled loss: bf16 or full precision)
        c.update(S=_loguniform(rng, 1, 32), L=_loguniform(rng, 1, 4096),
                 dtype=rng.choice(("f32", "bf16", "bf16") if kind == "train" else ("f32", "bf16", "bf16", "f16")),
                 fused=rng.random() < 0.5)
        pairs = c["S"] * c["L"] ** 2 * c["H"] * (8 if c["dtype"] == "f32" else 1)
        if c["H"] <= 64 and pairs * c["D"] <= 4 * 4096 ** 2 * 32 * 128 and pairs <= 4 * 4096 ** 2 * 32:
            return c


def _lengths(case):
    """The lengths that a case's sequences have: the longest, and others from an
    eighth of it on; one of several is of none where the case has an empty place."""
    r = random.Random("%d %d" % (case["S"], case["L"]))
    lens = [case["L"]] + [max(1, int(case["L"] * r.uniform(0.125, 1.0))) for _ in range(case["S"] - 1)]
    r.shuffle(lens)
    if case["empty"] and len(lens) > 1:
        lens[len(lens) // 2] = 0
    return lens


def _pages_of(case):
    return -(-case["L"] // case["P"])


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, sd=1.0):
        return (torch.randn(shape, generator=g, device=dev) * sd).to(t)

    st = dict(case, scale=1.0 / math.sqrt(case["D"]))
    HK, D = case["HK"], case["D"]
    if case["kind"] in ("prompt", "train"):
        lens, H = _lengths(case), case["H"]
        N = max(1, sum(lens))
        cu = torch.zeros(case["S"] + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(lens).cumsum(0).to(torch.int32)
        st.update(cu=cu.to(dev), L=max(lens), N=N)
        if case["fused"]:
            qkv = normal(N, (H + 2 * HK) * D)
            q, k, v = qkv.split((H * D, HK * D, HK * D), 1)
            st.update(q=q.view(N, H, D), k=k.view(N, HK, D), v=v.view(N, HK, D))
        else:
            st.update(q=normal(N, H, D), k=normal(N, HK, D), v=normal(N, HK, D))
        if case["kind"] == "train":
            st.update(do=normal(N, H, D, sd=0.05))
        return st
    if case["kind"] == "cache":
        N, P, pages, c = case["N"], case["P"], case["pages"], _TYPES[case["cache"]]
        if case["fused"]:
            k, v = normal(N, 2 * HK * D).split((HK * D, HK * D), 1)
            st.update(k=k.view(N, HK, D), v=v.view(N, HK, D))
        else:
            st.update(k=normal(N, HK, D), v=normal(N, HK, D))
        # a prompt takes whole pages in any order, a step one row of each of many
        if N < pages:
            page = torch.randperm(pages, generator=g, device=dev)[:N]
            slots = page * P + torch.randint(0, P, (N,), generator=g, device=dev)
        else:
            page = torch.randperm(pages, generator=g, device=dev)[:-(-N // P)]
            slots = (page[:, None] * P + torch.arange(P, device=dev)).reshape(-1)[:N]
        st.update(slots=slots.contiguous())
        for name in ("k", "v"):
            st[name + "_cache"] = torch.zeros(pages, HK, P, D, dtype=c, device=dev)
            st[name + "_scale"] = torch.zeros(pages, HK, P, device=dev) if case["cache"] == "i8" else None
        return st
    lens, P, H, per = _lengths(case), case["P"], case["H"], _pages_of(case)
    used = [-(-n // P) for n in lens]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table, at = torch.full((case["S"], per), -1, dtype=torch.int32, device=dev), 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    st.update(q=normal(case["S"], H, D), table=table, lens=torch.tensor(lens, dtype=torch.int32).to(dev), L=max(lens))
    for name in ("k", "v"):
        x = normal(pages, HK, P, D)
        st[name + "_scale"] = None
        if case["cache"] == "i8":
            scale = _row_scale(x)
            st[name + "_scale"] = scale.contiguous()
            x = (x.float() / scale[..., None]).round().clamp(-127, 127).to(torch.int8)
        st[name + "_cache"] = x
    return st


# ------------------------------------------------------------------ plain forms

def _row_scale(x):
    """A row's scale in an 8-bit cache: its largest magnitude becomes 127.  (Divided
    in 64 bits: in 32, torch multiplies by a reciprocal on the GPU.)"""
    return (x.abs().amax(-1).double() / 127.0).float().clamp_min(2.0 ** -126)


def _padded(st):
    """The packed rows of each sequence [S][L], and each packed row's place there."""
    cu, N, S, L = st["cu"].long(), st["N"], st["S"], st["L"]
    rows = torch.arange(N, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), rows, right=True).clamp_max(S - 1)
    at = (cu[:-1, None] + torch.arange(L, device=cu.device)).clamp_max(N - 1)
    return at, seq, (rows - cu[seq]).clamp_max(L - 1)


def _heads(x, at, G):
    """[N][heads][D] -> [S * kv heads][G * L][D] in 32 bits, the G heads of a group one after the other."""
    S, L = at.shape
    H, D = x.shape[1:]
    x = x.float()[at].view(S, L, H // G, G, D).permute(0, 2, 3, 1, 4)
    return x.reshape(S * (H // G), G * L, D)


def _unheads(x, S, G, L, seq, pos):
    """The inverse of _heads for the packed rows."""
    HK, D = x.shape[0] // S, x.shape[-1]
    x = x.view(S, HK, G, L, D).permute(0, 3, 1, 2, 4).reshape(S, L, HK * G, D)
    return x[seq, pos]


def _plain_forward(st):
    S, L, HK, G = st["S"], st["L"], st["HK"], st["H"] // st["HK"]
    at, seq, pos = _padded(st)
    q, k, v = _heads(st["q"], at, G), _heads(st["k"], at, 1), _heads(st["v"], at, 1)
    s = torch.matmul(q, k.transpose(1, 2)).mul_(st["scale"])
    later = torch.ones(L, L, dtype=torch.bool, device=s.device).triu_(1)
    s.view(S * HK, G, L, L).masked_fill_(later, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / l
    lse = _unheads(m + l.log(), S, G, L, seq, pos)[..., 0].t().contiguous()
    return (at, seq, pos), (q, k, v, o), p.div_(l), lse


def _plain_prompt(st):
    (_, seq, pos), (_, _, _, o), _, lse = _plain_forward(st)
    o = _unheads(o, st["S"], st["H"] // st["HK"], st["L"], seq, pos)
    return {"o": o.to(st["q"].dtype), "lse": lse}


def _plain_train(st):
    S, L, G, t = st["S"], st["L"], st["H"] // st["HK"], st["q"].dtype
    (at, seq, pos), (q, k, v, o), p, lse = _plain_forward(st)
    # rows past a sequence's end repeat others: they give nothing
    inside = torch.arange(L, device=p.device) < (st["cu"][1:] - st["cu"][:-1])[:, None]
    do = _heads(st["do"], at, G).view(S, -1, G, L, st["D"]) * inside[:, None, None, :, None]
    do = do.reshape(q.shape)
    dv = torch.matmul(p.transpose(1, 2), do)
    ds = torch.matmul(do, v.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(st["scale"])
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q)

    def rows(x, G):
        return _unheads(x, S, G, L, seq, pos).to(t)

    return {"o": rows(o, G), "lse": lse, "dq": rows(dq, G), "dk": rows(dk, 1), "dv": rows(dv, 1)}


def _plain_cache(st):
    P, slots, out = st["P"], st["slots"], {}
    page, off = slots // P, slots % P
    for name in ("k", "v"):
        x, cache, scales = st[name], st[name + "_cache"], st[name + "_scale"]
        if scales is None:
            cache[page, :, off] = x.to(cache.dtype)
            out[name] = cache[page, :, off].to(x.dtype)
        else:
            scale = _row_scale(x)
            # in 64 bits: values next to the border between two steps
            cache[page, :, off] = (x.double() / scale.double()[..., None]).round().clamp(-127, 127).to(torch.int8)
            scales[page, :, off] = scale
            out[name] = (cache[page, :, off].float() * scales[page, :, off][..., None]).to(x.dtype)
            out[name + "_scale"] = scales
    if st["k_scale"] is None:
        out.update(k_cache=st["k_cache"], v_cache=st["v_cache"])
    return out


def _plain_decode(st):
    S, H, D = st["q"].shape
    HK, P, L = st["HK"], st["P"], st["L"]
    table = st["table"].long().clamp_min(0)
    kv = []
    for name in ("k", "v"):
        x = st[name + "_cache"][table].float()  # [S][pages][HK][P][D]
        if st[name + "_scale"] is not None:
            x *= st[name + "_scale"][table][..., None]
        kv.append(x.transpose(1, 2).reshape(S * HK, -1, D))
    q = st["q"].float().view(S * HK, H // HK, D)
    s = torch.matmul(q, kv[0].transpose(1, 2)).mul_(st["scale"]).view(S, H, -1)
    there = torch.arange(s.shape[-1], device=s.device) < st["lens"][:, None, None]
    s = s.masked_fill(~there, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = (s - m).exp()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S * HK, H // HK, -1), kv[1]).view(S, H, D) / l.clamp_min(1e-38)
    lse = torch.where(l > 0, m + l.log(), -math.inf)[..., 0]
    return {"o": o.to(st["q"].dtype), "lse": lse}


def run(st):
    kind = st["kind"]
    if own:
        wha = _wha()
        if kind == "prompt":
            o, lse = wha.packed_fwd(st["q"], st["k"], st["v"], st["cu"])
            return {"o": o, "lse": lse}
        if kind == "train":
            q, k, v = st["q"], st["k"], st["v"]
            o, lse = wha.packed_fwd(q, k, v, st["cu"])
            grads = (None, None, None)
            if st["fused"]:  # the gradient of the fused projection's rows, in place
                (N, H, D), HK = q.shape, k.shape[1]
                dqkv = torch.empty(N, (H + 2 * HK) * D, dtype=q.dtype, device=q.device)
                x = dqkv.split((H * D, HK * D, HK * D), 1)
                grads = (x[0].view(N, H, D), x[1].view(N, HK, D), x[2].view(N, HK, D))
            dq, dk, dv = wha.packed_bwd(q, k, v, o, st["do"], lse, st["cu"], dq=grads[0], dk=grads[1], dv=grads[2])
            return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
        if kind == "cache":
            pages = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
            wha.paged_kv_write(st["k"], st["v"], st["slots"], *pages)
            k, v = wha.paged_kv_read(st["slots"], *pages, dtype=st["k"].dtype)
            if st["k_scale"] is None:
                return {"k": k, "v": v, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
            return {"k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
        o, lse = wha.paged_decode_fwd(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                                      k_scale=st["k_scale"], v_scale=st["v_scale"], want_lse=True)
        return {"o": o, "lse": lse}
    if kind == "prompt":
        return _plain_prompt(st)
    if kind == "train":
        return _plain_train(st)
    if kind == "cache":
        return _plain_cache(st)
    return _plain_decode(st)


# ------------------------------------------------------------------ least work

def work(case):
    size, HK, D = _SIZE[case["dtype"]], case["HK"], case["D"]
    if case["kind"] == "cache":
        rows = 2 * case["N"] * HK  # of k and of v
        cached = D * _SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0)
        # written: read the rows, write the cache; read back: the other way round
        return {"bytes": 2 * rows * (D * size + cached) + 2 * 8 * case["N"],
                "flops": 6 * rows * D if case["cache"] == "i8" else 0}
    lens, H = _lengths(case), case["H"]
    n = sum(lens)
    if case["kind"] == "decode":
        row = D * _SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0)
        pages = sum(-(-x // case["P"]) for x in lens)
        return {"bytes": 2 * n * HK * row + 2 * case["S"] * H * D * size + 4 * case["S"] * H + 4 * (pages + case["S"]),
                "flops": 4 * n * H * D}
    pairs = sum(x * (x + 1) // 2 for x in lens) * H
    qo, kv, lse = n * H * D * size, n * HK * D * size, 4 * n * H
    if case["kind"] == "prompt":
        return {"bytes": 2 * qo + 2 * kv + lse, "flops": 4 * pairs * D}
    # q, k, v and do read once, o, lse, dq, dk and dv written once
    return {"bytes": 4 * qo + 4 * kv + lse, "flops": 12 * pairs * D}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """One sequence and one group of heads after the other, in 64 bits."""
    st = prepare(case, seed)
    if case["kind"] == "cache":
        return _exact_cache(st)
    return _exact_decode(st) if case["kind"] == "decode" else _exact_packed(st)


def _exact_packed(st):
    G, q = st["H"] // st["HK"], st["q"]
    N, H, D = q.shape
    out = {"o": torch.zeros(N, H, D, dtype=torch.float64, device=q.device),
           "lse": torch.zeros(H, N, dtype=torch.float64, device=q.device)}
    train = st["kind"] == "train"
    if train:
        out.update({"d" + n: torch.zeros(st[n].shape, dtype=torch.float64, device=q.device) for n in "qkv"})
    bounds = st["cu"].tolist()
    for a, b in zip(bounds[:-1], bounds[1:]):
        for h in range(H if b > a else 0):
            qh, kh, vh = st["q"][a:b, h].double(), st["k"][a:b, h // G].double(), st["v"][a:b, h // G].double()
            s = (qh @ kh.T) / math.sqrt(D)
            s = s.tril() + torch.full_like(s, -math.inf).triu(1)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            o = p @ vh
            out["o"][a:b, h], out["lse"][h, a:b] = o, lse
            if train:
                do = st["do"][a:b, h].double()
                dp = do @ vh.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
                out["dq"][a:b, h] = ds @ kh
                out["dk"][a:b, h // G] += ds.T @ qh
                out["dv"][a:b, h // G] += p.T @ do
    return out


def _exact_cache(st):
    out = {}
    for name in ("k", "v"):
        x = st[name].double()
        HK, P = x.shape[1], st["P"]
        # a slot's rows as they lie: (page, head, place)
        page = torch.div(st["slots"], P, rounding_mode="floor")
        flat = (page[:, None] * HK + torch.arange(HK, device=x.device)) * P + (st["slots"] - page * P)[:, None]
        cache = st[name + "_cache"]
        if st[name + "_scale"] is None:
            whole = torch.zeros(cache.shape, dtype=torch.float64, device=x.device)
            whole.view(-1, x.shape[-1]).index_copy_(0, flat.reshape(-1), x.reshape(-1, x.shape[-1]))
            out[name], out[name + "_cache"] = x, whole
        else:
            # the scale is kept in 32 bits, and what a step stands for goes by that
            scale = (torch.maximum(x.amax(-1), -x.amin(-1)) / 127).clamp_min(2.0 ** -126).float().double()
            scales = torch.zeros(st[name + "_scale"].shape, dtype=torch.float64, device=x.device)
            scales.view(-1).index_copy_(0, flat.reshape(-1), scale.reshape(-1))
            out[name] = torch.round(x / scale.unsqueeze(-1)) * scale.unsqueeze(-1)
            out[name + "_scale"] = scales
    return out


def _exact_decode(st):
    S, H, D = st["q"].shape
    G = H // st["HK"]
    o = torch.zeros(S, H, D, dtype=torch.float64, device=st["q"].device)
    lse = torch.full((S, H), -math.inf, dtype=torch.float64, device=o.device)
    for i, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        ids = st["table"][i, :-(-n // st["P"])].long()
        rows = []
        for name in ("k", "v"):
            x = st[name + "_cache"].index_select(0, ids).double()
            if st[name + "_scale"] is not None:
                x = x * st[name + "_scale"].index_select(0, ids).double().unsqueeze(-1)
            rows.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n])
        for h in range(H):
            s = rows[0][h // G] @ st["q"][i, h].double() / math.sqrt(D)
            lse[i, h] = torch.logsumexp(s, 0)
            o[i, h] = torch.exp(s - lse[i, h]) @ rows[1][h // G]
    return {"o": o, "lse": lse}
