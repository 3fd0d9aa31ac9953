"""The paged key-value cache: rows written (as they are, or in 8 bits) and read
back, and the attention of one new token over it, against 64 bits."""
import math

import pytest
import torch

from packed_reference import decode, near, quantise

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def empty_cache(pages, HK, P, D, dtype, fill=0):
    kv = [torch.full((pages, HK, P, D), fill, dtype=dtype, device=DEV) for _ in range(2)]
    sc = [torch.full((pages, HK, P), float("nan"), device=DEV) if dtype == I8 else None for _ in range(2)]
    return kv + sc


def at(cache, slots, P):
    """The rows [N][HK] of slots."""
    return cache[slots // P, :, slots % P]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("N,HK,P,D,fused,off", [(1, 1, 1, 64, False, 0), (7, 3, 16, 64, True, 0),
                                               (200, 8, 64, 128, True, 0), (65, 2, 4096, 42, False, 0),
                                               (33, 4, 8, 100, True, 0), (50, 2, 2, 128, False, 1),
                                               (19, 1, 32, 1, False, 0), (40, 5, 128, 40, True, 3)])
def test_write_and_read(pkg, dtype, eight, N, HK, P, D, fused, off):
    print(f"paged write {dtype} eight={eight} N={N} HK={HK} P={P} D={D}", flush=True)
    g = gen(N + D)
    if fused:
        x = torch.randn(N * 2 * HK * D + off, generator=g, device=DEV).to(dtype)[off:].view(N, 2 * HK * D)
        k, v = (t.view(N, HK, D) for t in x.split((HK * D, HK * D), 1))
    else:
        k, v = (torch.randn(N * HK * D + off, generator=g, device=DEV).to(dtype)[off:].view(N, HK, D) for _ in range(2))
    pages = -(-N // P) + 2
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:N]
    cache = empty_cache(pages, HK, P, D, I8 if eight else dtype, 3)
    before = [t.clone() if t is not None else None for t in cache]
    pkg.paged_kv_write(k, v, slots, *cache)
    for x, c, s, c0, s0 in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        if eight:
            codes, scales = quantise(x)
            assert torch.equal(at(c, slots, P), codes) and torch.equal(at(s, slots, P), scales)
            s0[slots // P, :, slots % P] = scales
            assert torch.equal(s.nan_to_num(-1.0), s0.nan_to_num(-1.0))
            c0[slots // P, :, slots % P] = codes
        else:
            c0[slots // P, :, slots % P] = x
        assert torch.equal(c, c0)  # every other place as it was
    for out in (dtype, F32) if eight else (dtype,):
        rk, rv = pkg.paged_kv_read(slots, *cache, dtype=out)
        for x, r, s, c in ((k, rk, cache[2], cache[0]), (v, rv, cache[3], cache[1])):
            want = (at(c, slots, P).float() * at(s, slots, P)[..., None]).to(out) if eight else x
            assert r.dtype == out and torch.equal(r, want)
            if eight:  # half a step of the row, and the rounding of the answer
                step = at(s, slots, P)[..., None]
                assert bool(((r.float() - x.float()).abs() <= step * 0.50001 + x.float().abs() * torch.finfo(out).eps).all())


def test_steps_at_their_borders(pkg):
    """Ties, the largest and smallest magnitudes, zeros, infinities and NaN in a row of an 8-bit cache."""
    D, rows = 64, []
    half = torch.arange(D, device=DEV).float() - 31.5
    rows.append(torch.cat([half[:-1], torch.tensor([127.0], device=DEV)]))          # scale 1: x.5 to the even step
    rows.append(torch.cat([3 * half[:-1], torch.tensor([-381.0], device=DEV)]))     # scale 3: ties of a scale that is no power of two
    rows.append(torch.zeros(D, device=DEV))
    rows.append(torch.full((D,), 1e-40, device=DEV))
    rows.append(torch.full((D,), 3.0e38, device=DEV) * torch.linspace(-1, 1, D, device=DEV))
    rows.append(torch.linspace(-1, 1, D, device=DEV) * 1e-37)
    x = torch.stack(rows)[:, None]
    n = x.shape[0]
    cache = empty_cache(2, 1, 8, D, I8)
    slots = torch.arange(n, device=DEV)
    pkg.paged_kv_write(x, x, slots, *cache)
    codes, scales = quantise(x)
    assert torch.equal(at(cache[0], slots, 8), codes) and torch.equal(at(cache[2], slots, 8), scales)
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        y[1, 0, 5] = bad
        pkg.paged_kv_write(y, x, slots, *cache)
        k, v = pkg.paged_kv_read(slots, *cache)
        assert bool(torch.isnan(k[1]).all()) and bool(torch.isfinite(k[[0, 2, 3, 4, 5]]).all()) and bool(torch.isfinite(v).all())


def test_slots_outside_the_cache(pkg):
    """Negative slots and ones past the last page: nothing written, zeros read; a slot read twice."""
    for dtype in (BF16, I8):
        g = gen(3)
        around = empty_cache(10, 2, 16, 64, dtype, 1)
        cache = [t[3:7] if t is not None else None for t in around]
        k, v = (torch.randn(6, 2, 64, generator=g, device=DEV).to(BF16) for _ in range(2))
        slots = torch.tensor([-1, 5, 64, -(2 ** 40), 2 ** 40, 63], device=DEV)
        before = [t.clone() if t is not None else None for t in around]
        pkg.paged_kv_write(k, v, slots, *cache)
        for a, b in zip(around, before):
            if a is not None:
                b[3, :, 5], b[6, :, 15] = a[3, :, 5], a[6, :, 15]
                assert torch.equal(a.float().nan_to_num(-9.0), b.float().nan_to_num(-9.0))
        rk, rv = pkg.paged_kv_read(torch.cat([slots, slots[1:2], slots[1:2]]), *cache, dtype=BF16)
        for i in (0, 2, 3, 4):
            assert not bool(rk[i].any()) and not bool(rv[i].any())
        assert torch.equal(rk[1], rk[6]) and torch.equal(rk[1], rk[7]) and bool(rk[1].any()) and bool(rv[5].any())


def make(lens, H, HK, P, D, dtype, eight, seed, spare=3, extra=0):
    g = gen(seed)
    used = [max(0, -(-n // P)) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    per = max(1, max(used)) + extra
    table, i = torch.full((len(lens), per), -7, dtype=torch.int32, device=DEV), 0
    for b, n in enumerate(used):
        table[b, :n] = order[i:i + n]
        i += n
    q = torch.randn(len(lens), H, D, generator=g, device=DEV).to(dtype)
    kv, sc = [], []
    for _ in range(2):
        x = torch.randn(pages, HK, P, D, generator=g, device=DEV).to(dtype)
        codes, scales = quantise(x) if eight else (x, None)
        kv.append(codes.contiguous())
        sc.append(scales.contiguous() if eight else None)
    return q, kv, sc, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def run(pkg, q, kv, sc, table, lens, **kw):
    return pkg.paged_decode_fwd(q, kv[0], kv[1], table, lens, k_scale=sc[0], v_scale=sc[1], want_lse=True, **kw)


def check(pkg, lens, H, HK, P, D, dtype, eight, seed=1, **kw):
    print(f"paged decode {dtype} eight={eight} lens={lens} H={H} HK={HK} P={P} D={D}", flush=True)
    q, kv, sc, table, ln = make(lens, H, HK, P, D, dtype, eight, seed, **kw)
    # what lies behind a sequence's last position may be anything
    for b, n in enumerate(lens):
        if n > 0 and n % P:
            page = int(table[b, n // P])
            for c, s in zip(kv, sc):
                if s is not None:
                    s[page, :, n % P:] = float("nan")
                else:
                    c[page, :, n % P:] = float("nan")
    o, lse = run(pkg, q, kv, sc, table, ln)
    ref = decode(q, kv[0], kv[1], table, lens, pkg.default_scale(D), sc[0], sc[1])
    near("o", o, ref["o"])
    empty = [b for b, n in enumerate(lens) if n <= 0]
    full = [b for b, n in enumerate(lens) if n > 0]
    near("lse", lse[full], [x[full] for x in ref["lse"]])
    assert not bool(o[empty].any()) and bool((lse[empty] == -math.inf).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lens,P", [([1], 16), ([0, 1, 2, 31, 32, 33, 63, 64, 65], 16), ([127, 129, 0, 1000], 32),
                                    ([40, 3], 1), ([300, 77, 500], 8), ([4095, 4097], 4096), ([3000, 1, 2222], 64)])
def test_lengths(pkg, lens, P, dtype, eight):
    check(pkg, lens, 4, 2, P, 64, dtype, eight)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("H,HK,D", [(2, 2, 128), (8, 1, 128), (16, 1, 64), (17, 1, 64), (64, 2, 128), (12, 4, 64),
                                    (4, 4, 42), (3, 1, 100), (6, 2, 40), (1, 1, 1), (5, 5, 127), (10, 2, 8)])
def test_heads_and_dims(pkg, H, HK, D, dtype, eight):
    check(pkg, [130, 0, 1, 700], H, HK, 32, D, dtype, eight, extra=5)


@pytest.mark.parametrize("eight", [False, True])
def test_long_cache_is_split_and_joined(pkg, eight):
    check(pkg, [40000, 5, 12345], 8, 2, 64, 128, BF16, eight, seed=5)
    check(pkg, [100003], 4, 1, 16, 64, F32 if not eight else F16, eight, seed=6)


@pytest.mark.parametrize("eight", [False, True])
def test_bad_tables_give_nan_for_their_sequence_only(pkg, eight):
    """A page outside the cache below the length, and a length past the table: NaN, the others keep their bits."""
    for P, lens in ((16, [100, 40, 64, 20]), (64, [9000, 3000, 8000, 100])):
        q, kv, sc, table, ln = make(lens, 4, 2, P, 64, BF16, eight, 7, extra=2)
        want, want_lse = run(pkg, q, kv, sc, table, ln)
        for bad in (-1, kv[0].shape[0], 2 ** 31 - 1, -2 ** 31):
            t = table.clone()
            t[0, 1], t[2, 0] = bad, bad
            o, lse = run(pkg, q, kv, sc, t, ln)
            for b in (0, 2):
                assert bool(torch.isnan(o[b]).all()) and bool(torch.isnan(lse[b]).all())
            for b in (1, 3):
                assert torch.equal(o[b], want[b]) and torch.equal(lse[b], want_lse[b])
        longer = ln.clone()
        longer[1] = table.shape[1] * P + 1
        t = table.clamp_min(0)
        o, lse = run(pkg, q, kv, sc, t, longer)
        assert bool(torch.isnan(o[1]).all()) and bool(torch.isnan(lse[1]).all())
        assert torch.equal(o[3], want[3])
        longer[1] = 2 ** 31 - 1
        longer[0] = -3
        o, lse = run(pkg, q, kv, sc, t, longer)
        assert bool(torch.isnan(o[1]).all()) and not bool(o[0].any()) and bool((lse[0] == -math.inf).all())


def test_shared_pages_and_strided_queries(pkg):
    """Two sequences that share their first pages (a common prompt), q and o as slices of wider rows."""
    q, kv, sc, table, ln = make([100, 90], 4, 2, 16, 64, BF16, False, 8)
    table[1, :4] = table[0, :4]
    wide = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(9)).to(BF16)
    out = torch.zeros(2, 4, 100, dtype=BF16, device=DEV)
    o, lse = run(pkg, wide[:, 1], kv, sc, table, ln, out=out[..., :64])
    ref = decode(wide[:, 1], kv[0], kv[1], table, [100, 90], pkg.default_scale(64))
    near("o", o, ref["o"])
    near("lse", lse, ref["lse"])
    assert not bool(out[..., 64:].any())


def test_unaligned_cache_and_queries(pkg):
    q, kv, sc, table, ln = make([100, 9], 4, 2, 16, 64, BF16, False, 10)
    odd = [torch.cat([c.flatten()[:1], c.flatten()])[1:].view(c.shape) for c in kv]
    q2 = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)
    o, lse = run(pkg, q2, odd, sc, table, ln)
    ref = decode(q, kv[0], kv[1], table, [100, 9], pkg.default_scale(64))
    near("o", o, ref["o"])
    near("lse", lse, ref["lse"])


def test_cache_past_32_bits(pkg):
    """Pages whose rows lie past 2^32 bytes and 2^31 elements."""
    HK, P, D = 8, 256, 128
    pages = (2 ** 31) // (HK * P * D) + 40
    kv = [torch.zeros(pages, HK, P, D, dtype=BF16, device=DEV) for _ in range(2)]
    g = gen(11)
    last = torch.arange(pages - 8, pages, device=DEV)
    k, v = (torch.randn(8 * P, HK, D, generator=g, device=DEV).to(BF16) for _ in range(2))
    slots = (last[:, None] * P + torch.arange(P, device=DEV)).flatten()
    pkg.paged_kv_write(k, v, slots, *kv)
    rk, rv = pkg.paged_kv_read(slots, *kv)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    table = last.flip(0).to(torch.int32)[None].contiguous()
    q = torch.randn(1, 16, D, generator=g, device=DEV).to(BF16)
    ln = torch.tensor([8 * P - 5], dtype=torch.int32, device=DEV)
    o, lse = run(pkg, q, kv, [None, None], table, ln)
    ref = decode(q, kv[0], kv[1], table, [8 * P - 5], pkg.default_scale(D))
    near("o", o, ref["o"])
    near("lse", lse, ref["lse"])


@pytest.mark.parametrize("dtype,eight", [(BF16, False), (BF16, True), (F32, False)])
def test_not_finite_rows(pkg, dtype, eight):
    """NaN in a cached row reaches its own sequence and heads, an infinite value row its columns."""
    q, kv, sc, table, ln = make([90, 50], 4, 2, 16, 64, dtype, eight, 12)
    want, _ = run(pkg, q, kv, sc, table, ln)
    page, place = int(table[0, 2]), 3
    c = sc[0] if eight else kv[0]
    c[page, 0, place] = float("nan")
    o, lse = run(pkg, q, kv, sc, table, ln)
    assert bool(torch.isnan(o[0, :2]).all()) and bool(torch.isnan(lse[0, :2]).all())
    assert torch.equal(o[0, 2:], want[0, 2:]) and torch.equal(o[1], want[1])
    if not eight:
        c[page, 0, place] = 0.0
        kv[1][page, 0, place, 7] = float("inf")
        o, lse = run(pkg, q, kv, sc, table, ln)
        assert bool((o[0, :2, 7] == math.inf).all()) and bool(torch.isfinite(o[0, :2, :7]).all())


def test_serving_run(pkg):
    """A prompt's attention, its rows into an 8-bit cache, then steps that write a token and attend to all so far;
    one graph of the step, replayed as the cache grows; against 64 bits over the rows that the cache stands for."""
    H, HK, D, P, steps = 8, 2, 64, 16, 20
    lens, g = [37, 5, 64], gen(21)
    N = sum(lens)
    x = torch.randn(N, (H + 2 * HK) * D, generator=g, device=DEV).to(BF16)
    q, k, v = (t.view(N, -1, D) for t in x.split((H * D, HK * D, HK * D), 1))
    cu = torch.tensor([0, 37, 42, 106], dtype=torch.int32, device=DEV)
    o, _ = pkg.packed_fwd(q, k, v, cu)
    cache = empty_cache(40, HK, P, D, I8)
    table = torch.randperm(40, generator=g, device=DEV)[:30].view(3, 10).to(torch.int32)

    def slot(b, i):
        return table[b, i // P].long() * P + i % P

    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    seq = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(lens, device=DEV))
    pkg.paged_kv_write(k, v, slot(seq, pos), *cache)
    rk, rv = pkg.paged_kv_read(slot(seq, pos), *cache, dtype=BF16)
    # the last row of every prompt over the cache as the decode of a cache of its length
    last = cu[1:].long() - 1
    od, _ = run(pkg, q[last].contiguous(), cache[:2], cache[2:], table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    # 8-bit rows are off by at most max|row| / 254 of about 3: scores by 0.012 x 8 and values by 0.012
    assert float((od.float() - o[last].float()).abs().max()) <= 0.25
    assert float((rk.float() - k.float()).abs().max()) <= 0.5 * float(k.float().abs().max()) / 127 + 0.02

    sq, sk, sv = (torch.zeros(3, h, D, dtype=BF16, device=DEV) for h in (H, HK, HK))
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = torch.empty_like(sq), torch.empty(3, H, device=DEV)
    rows = torch.arange(3, device=DEV)

    def step():
        pkg.paged_kv_write(sk, sv, slot(rows, lengths.long()), *cache)
        lengths.add_(1)
        run(pkg, sq, cache[:2], cache[2:], table, lengths, out=out, lse=lse)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        lengths.sub_(1)
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    now = list(lens)
    for i in range(steps):
        for t in (sq, sk, sv):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        now = [n + 1 for n in now]
        assert lengths.tolist() == now
        ref = decode(sq, cache[0], cache[1], table, now, pkg.default_scale(D), cache[2], cache[3])
        near("o", out, ref["o"])
        near("lse", lse, ref["lse"])
        eager, _ = run(pkg, sq, cache[:2], cache[2:], table, lengths)
        assert torch.equal(eager, out)


def test_two_graphs_with_one_workspace(pkg):
    """Two captured calls that share a caller's workspace, replayed one after the other on one stream."""
    cases = [make(lens, 8, 2, 16, 64, BF16, False, 30 + i) for i, lens in enumerate(([9000, 100], [70, 8000]))]
    ws = torch.empty(8 << 20, dtype=torch.uint8, device=DEV)
    want = [run(pkg, *c) for c in cases]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c in cases:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(run(pkg, *c, workspace=ws))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
        ws.fill_(255)


def test_python_refusals_on_the_device(pkg):
    q, kv, sc, table, ln = make([100, 9], 4, 2, 16, 64, BF16, True, 13)
    k = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    slots = torch.arange(3, device=DEV)
    for bad in (lambda: pkg.paged_kv_write(k, k, slots, kv[0], kv[1]), lambda: pkg.paged_kv_write(k, k, slots.int(), *kv, *sc),
                lambda: pkg.paged_kv_write(k, k, slots[:2], *kv, *sc), lambda: pkg.paged_kv_write(k[:, :1], k[:, :1], slots, *kv, *sc),
                lambda: pkg.paged_kv_write(k, k, slots, kv[0].transpose(1, 2), kv[1].transpose(1, 2), *sc),
                lambda: pkg.paged_kv_read(slots, *kv, sc[0][:1], sc[1]),
                lambda: run(pkg, q, kv, sc, table.long(), ln), lambda: run(pkg, q, kv, sc, table, ln[:1]),
                lambda: run(pkg, q[..., :32], kv, sc, table, ln)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg.WaveHipError, match="workspace"):
        big = make([9000, 9], 4, 2, 16, 64, BF16, True, 13)
        run(pkg, *big, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(pkg.WaveHipError, match="cache_dtype"):
        run(pkg, q, [t.half() for t in kv], [None, None], table, ln)
