"""Attention of packed sequences with grouped heads, forward and backward,
against 64 bits (packed_reference.py derives the bounds)."""
import numpy as np
import pytest
import torch

from packed_reference import near, packed

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(lens, H, HK, D, dtype, seed, fused=False, tail=0, off=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    N = max(1, sum(lens)) + tail
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    if fused:
        W = (H + 2 * HK) * D
        x = torch.randn(N * W + off, generator=g, device=DEV).to(dtype)[off:].view(N, W)
        q, k, v = x.split((H * D, HK * D, HK * D), 1)
        q, k, v = q.view(N, H, D), k.view(N, HK, D), v.view(N, HK, D)
    else:
        q, k, v = (torch.randn(N * h * D + off, generator=g, device=DEV).to(dtype)[off:].view(N, h, D)
                   for h in (H, HK, HK))
    do = torch.randn(N, H, D, generator=g, device=DEV).to(dtype)
    return q, k, v, do, cu


def check(pkg, lens, H, HK, D, dtype, seed=1, bwd=True, scale=None, **kw):
    print(f"packed {dtype} lens={lens} H={H} HK={HK} D={D} {kw}", flush=True)
    q, k, v, do, cu = make(lens, H, HK, D, dtype, seed, **kw)
    o, lse = pkg.packed_fwd(q, k, v, cu, scale=scale)
    bwd = bwd and dtype != F16
    ref = packed(q, k, v, cu.tolist(), pkg.default_scale(D) if scale is None else scale, do if bwd else None)
    n = sum(lens)
    near("o", o, ref["o"], n)
    near("lse", lse, ref["lse"], n)
    if bwd:
        for name, x in zip(("dq", "dk", "dv"), pkg.packed_bwd(q, k, v, o, do, lse, cu, scale=scale)):
            near(name, x, ref[name], n)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [0, 5, 0, 64, 65, 0], [31, 32, 33], [127, 128, 129],
                                  [33, 200, 1, 0, 17], [700, 260]])
def test_lengths(pkg, lens, dtype):
    check(pkg, lens, 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H,HK,D", [(2, 2, 128), (8, 2, 128), (4, 4, 42), (6, 2, 40), (3, 1, 96), (5, 5, 100),
                                    (12, 4, 64), (7, 1, 56), (2, 1, 1), (2, 2, 8), (3, 3, 32), (2, 1, 127),
                                    (20, 1, 64), (128, 1, 16)])
def test_heads_and_dims(pkg, H, HK, D, dtype):
    check(pkg, [70, 1, 150], H, HK, D, dtype, fused=H % 2 == 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_rows(pkg, dtype):
    check(pkg, [40, 77], 4, 2, 64, dtype, off=1)
    check(pkg, [40, 77], 3, 1, 128, dtype, off=3, fused=True)


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (BF16, 128)])
def test_long_rows_and_many_sequences(pkg, dtype, D):
    check(pkg, [2100], 2, 1, D, dtype, seed=3)
    check(pkg, [(7 * i) % 23 for i in range(300)], 2, 1, D, dtype, seed=4)  # more than 64 sequences, many empty


def test_scale_and_large_scores(pkg):
    check(pkg, [90, 130], 4, 2, 64, F32, scale=0.031)
    # scores of some hundred: every row's weight on few keys, the running maximum moves often
    q, k, v, do, cu = make([150, 64], 4, 2, 64, BF16, 9)
    q, k = q * 8, k * 8
    o, lse = pkg.packed_fwd(q, k, v, cu)
    ref = packed(q, k, v, cu.tolist(), pkg.default_scale(64))
    # fp32 sums of scores of magnitude S are off by about 64 2^-24 S (S up to 64 x 8 here): 2e-3 of each weight
    near("o", o, (ref["o"][0], ref["o"][1] + 2e-3), 214)
    near("lse", lse, (ref["lse"][0], ref["lse"][1] + 2e-3), 214)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_behind_the_last_sequence_stay(pkg, dtype):
    q, k, v, do, cu = make([30, 41], 4, 2, 64, dtype, 5, tail=150)
    for t in (q, k, v, do):
        t[71:] = float("nan")
    o = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    lse = torch.full((4, q.shape[0]), 7.0, device=DEV)
    pkg.packed_fwd(q, k, v, cu, out=o, lse=lse)
    grads = [torch.full(t.shape, 7.0, dtype=dtype, device=DEV) for t in (q, k, v)]
    pkg.packed_bwd(q, k, v, o, do, lse, cu, dq=grads[0], dk=grads[1], dv=grads[2])
    ref = packed(q, k, v, cu.tolist(), pkg.default_scale(64), do)
    for name, x in (("o", o), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        tail = x[:, 71:] if name == "lse" else x[71:]
        assert bool((tail == 7.0).all()), name
        near(name, x, ref[name], 71)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_not_finite_rows_reach_no_earlier_row(pkg, dtype, value, D):
    """One infinity or NaN in q, k, v or do of position 40 of the second of three
    sequences: earlier positions and the other sequences keep their values."""
    lens, at = [50, 90, 50], 50 + 40
    for which in range(4):
        q, k, v, do, cu = make(lens, 4, 2, D, dtype, 6)
        ref = packed(q, k, v, cu.tolist(), pkg.default_scale(D), do)
        (q, k, v, do)[which][at, 1, 3] = value
        o, lse = pkg.packed_fwd(q, k, v, cu)
        dq, dk, dv = pkg.packed_bwd(q, k, v, o, do, lse, cu)
        keep = torch.ones(190, dtype=torch.bool, device=DEV)
        keep[at:140] = False  # the position and those after it in its sequence
        others = keep.clone()
        others[50:140] = False  # dk and dv of earlier keys take part in later rows
        for name, x, rows in (("o", o, keep), ("dq", dq, keep), ("dk", dk, others), ("dv", dv, others)):
            near(name, x[rows], (ref[name][0][rows], ref[name][1][rows]))
        near("lse", lse[:, keep], (ref["lse"][0][:, keep], ref["lse"][1][:, keep]))
        if which == 2 and value != value:
            assert bool(torch.isnan(o[at:140, 2:, 3]).all())  # (head 1's group) and later rows do take it
        if which == 3 and value != value:
            assert bool(torch.isnan(dv[50:at + 1, 0, 3]).all())
            # keys after the row that holds it get nothing of it
            near("dv", dv[at + 1:140], (ref["dv"][0][at + 1:140], ref["dv"][1][at + 1:140]))
            near("dk", dk[at + 1:140], (ref["dk"][0][at + 1:140], ref["dk"][1][at + 1:140]))


@pytest.mark.parametrize("dtype,D", [(F32, 48), (BF16, 64), (BF16, 40), (BF16, 42)])
def test_enough_keys_for_the_larger_blocks(pkg, dtype, D):
    """8231 rows of 8 key-value heads; then with a NaN in one sequence, which the others do not see."""
    lens = [1100, 1, 700, 1300, 900, 1200, 800, 1250, 980]
    q, k, v, do, cu = make(lens, 8, 8, D, dtype, 14)
    ref = packed(q, k, v, cu.tolist(), pkg.default_scale(D), do)
    rest = torch.ones(sum(lens), dtype=torch.bool, device=DEV)
    for spoil in (False, True):
        if spoil:
            v[2000, 5, 7] = float("nan")
            rest[1801:3101] = False
        o, lse = pkg.packed_fwd(q, k, v, cu)
        for name, x in (("o", o),) + tuple(zip(("dq", "dk", "dv"), pkg.packed_bwd(q, k, v, o, do, lse, cu))):
            near(name, x[rest], (ref[name][0][rest], ref[name][1][rest]))
        near("lse", lse, ref["lse"])  # (no score holds it)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_values(pkg, dtype):
    """Values of 2^100 with gradients of 2^-100: the bounds are relative, and no part of a split falls
    below 2^-126 where it counts."""
    q, k, v, do, cu = make([90, 40], 4, 2, 64, dtype, 15)
    v, do = v * 2.0 ** 100, do * 2.0 ** -100
    o, lse = pkg.packed_fwd(q, k, v, cu)
    ref = packed(q, k, v, cu.tolist(), pkg.default_scale(64), do)
    near("o", o, ref["o"])
    for name, x in zip(("dq", "dk", "dv"), pkg.packed_bwd(q, k, v, o, do, lse, cu)):
        up = 2.0 ** 100 if name == "dv" else 1.0
        near(name, x.double() * up, (ref[name][0] * up, ref[name][1] * up))


def test_two_streams_at_once(pkg):
    """Calls that alternate between two streams, each with inputs of its own and no workspace passed."""
    sets = [make(lens, 6, 2, 64, BF16, 50 + i) for i, lens in enumerate(([900, 700], [500, 40, 1000]))]

    def both(q, k, v, do, cu):
        o, lse = pkg.packed_fwd(q, k, v, cu)
        return (o, lse) + pkg.packed_bwd(q, k, v, o, do, lse, cu)

    want = [both(*x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(both(*sets[i % 2]))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(x, want[i % 2])), i


def test_offsets_past_32_bits(pkg):
    """Rows 2^17 elements apart: the last sequence lies past 2^32 bytes and 2^31 elements."""
    N, W, D = 17000, 1 << 17, 64
    base = torch.zeros(N, W, dtype=BF16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    base[:, :4 * D] = torch.randn(N, 4 * D, generator=g, device=DEV).to(BF16)
    q, k, v = base[:, :2 * D].view(N, 2, D), base[:, 2 * D:3 * D].view(N, 1, D), base[:, 3 * D:4 * D].view(N, 1, D)
    do = torch.randn(N, 2, D, generator=g, device=DEV).to(BF16)
    cu = torch.tensor([0, 16700, 17000], dtype=torch.int32, device=DEV)
    o, lse = pkg.packed_fwd(q, k, v, cu)
    grad = torch.zeros_like(base)
    gq, gk, gv = (grad[:, a * D:b * D].view(N, b - a, D) for a, b in ((0, 2), (2, 3), (3, 4)))
    pkg.packed_bwd(q, k, v, o, do, lse, cu, dq=gq, dk=gk, dv=gv)
    sub = [t[16700:].contiguous() for t in (q, k, v, do)]
    ref = packed(*sub[:3], [0, 300], pkg.default_scale(D), sub[3])
    for name, x in (("o", o), ("dq", gq), ("dk", gk), ("dv", gv)):
        near(name, x[16700:], ref[name])
    near("lse", lse[:, 16700:], ref["lse"])


def test_cu_seqlens_that_do_not_fit_touch_nothing_else(pkg):
    """Entries outside [0, N], and ones that decrease: what lies around the outputs stays."""
    N, H, D = 70, 2, 64
    q, k, v, do, _ = make([N], H, 1, D, BF16, 8)
    for entries in ([0, N + 1000, 2 ** 31 - 1], [-5, 30, 2 ** 30], [0, 60, 10, 70], [70, 0, 70], [2 ** 30, 2 ** 30, 0]):
        cu = torch.tensor(entries, dtype=torch.int32, device=DEV)
        around = torch.full((N + 400, H, D), 5.0, dtype=BF16, device=DEV)
        grads = [torch.full((N + 400, h, D), 5.0, dtype=BF16, device=DEV) for h in (H, 1, 1)]
        stats = torch.full((3 * H, N), 5.0, device=DEV)
        pkg.packed_fwd(q, k, v, cu, out=around[200:200 + N], lse=stats[H:2 * H])
        inner = [g[200:200 + N] for g in grads]
        pkg.packed_bwd(q, k, v, around[200:200 + N], do, stats[H:2 * H], cu, dq=inner[0], dk=inner[1], dv=inner[2])
        torch.cuda.synchronize()
        for t in [around] + grads:
            assert bool((t[:200] == 5.0).all()) and bool((t[200 + N:] == 5.0).all()), entries
        assert bool((stats[:H] == 5.0).all()) and bool((stats[2 * H:] == 5.0).all()), entries


def test_same_bits_every_time_and_on_another_stream(pkg):
    q, k, v, do, cu = make([300, 17, 129], 6, 2, 64, BF16, 11)

    def once():
        o, lse = pkg.packed_fwd(q, k, v, cu)
        return (o, lse) + pkg.packed_bwd(q, k, v, o, do, lse, cu)

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_calls_follow_their_inputs(pkg):
    """Forward and backward in one graph, replayed on new inputs and other lengths, with eager work between."""
    lens = [[100, 60, 40], [1, 199, 0], [66, 67, 67]]
    q, k, v, do, cu = make(lens[0], 4, 2, 64, BF16, 20)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        pkg.packed_bwd(q, k, v, *(lambda o, l: (o, do, l))(*pkg.packed_fwd(q, k, v, cu)), cu)
        with torch.cuda.graph(graph, stream=stream):
            o, lse = pkg.packed_fwd(q, k, v, cu)
            grads = pkg.packed_bwd(q, k, v, o, do, lse, cu)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(6):
        new = make(lens[i % 3], 4, 2, 64, BF16, 30 + i)
        for a, b in zip((q, k, v, do, cu), new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want_o, want_lse = pkg.packed_fwd(*new[:3], new[4])
        want = pkg.packed_bwd(*new[:3], want_o, new[3], want_lse, new[4])
        for a, b in zip((o, lse) + grads, (want_o, want_lse) + want):
            assert torch.equal(a, b), i


def test_gradients_against_differences(pkg):
    """fp32 gradients of sum(o w) against central differences of the 64-bit formula along random directions."""
    lens, D = [19, 40], 32
    q, k, v, w, cu = make(lens, 4, 2, D, F32, 13)
    o, lse = pkg.packed_fwd(q, k, v, cu)
    grads = pkg.packed_bwd(q, k, v, o, w, lse, cu)
    g = torch.Generator(device=DEV).manual_seed(14)
    s = pkg.default_scale(D)
    for i in range(3):
        x = [q.double(), k.double(), v.double()]
        d = torch.randn(x[i].shape, generator=g, device=DEV, dtype=torch.float64)

        def value(eps):
            y = list(x)
            y[i] = x[i] + eps * d
            return float((packed(*y, cu.tolist(), s)["o"][0] * w.double()).sum())

        h = 1e-4  # third derivatives of order 10^2 here: the difference is off by about h^2 x 10^2 = 1e-6
        want = (value(h) - value(-h)) / (2 * h)
        got = float((grads[i].double() * d).sum())
        size = float((grads[i].double() * d).abs().sum())
        assert abs(got - want) <= 2e-5 * size + 1e-4, (i, got, want)


def test_equal_lengths_match_the_batched_operator(pkg):
    """The same numbers as [B,H,T,D] attention, up to fp32 rounding."""
    B, T, H, D = 3, 80, 4, 64
    q, k, v, do, cu = make([T] * B, H, H, D, F32, 15)
    o, lse = pkg.packed_fwd(q, k, v, cu)
    dq, dk, dv = pkg.packed_bwd(q, k, v, o, do, lse, cu)
    bh = [t.view(B, T, H, D).transpose(1, 2) for t in (q, k, v, do)]
    bo, bl = pkg.attn_fwd(*bh[:3])
    bg = pkg.attn_bwd(*bh[:3], bo, bh[3], bl)
    for a, b in zip((o, dq, dk, dv), (bo,) + bg):
        a = a.view(B, T, H, D).transpose(1, 2)
        assert float((a - b).norm() / b.norm()) <= 2e-6
    assert float((lse.view(H, B, T).transpose(0, 1) - bl).abs().max()) <= 1e-5


def test_python_refusals_on_the_device(pkg):
    q, k, v, do, cu = make([20], 4, 2, 64, BF16, 16)
    o, lse = pkg.packed_fwd(q, k, v, cu)
    for bad in (lambda: pkg.packed_fwd(q, k, v, cu.long()), lambda: pkg.packed_fwd(q, k[:, :1], v, cu),
                lambda: pkg.packed_fwd(q, k, v, cu, out=o[:, :2]), lambda: pkg.packed_fwd(q, k, v, cu.cpu()),
                lambda: pkg.packed_bwd(q, k, v, o, do.transpose(0, 1).contiguous().transpose(0, 1), lse, cu),
                lambda: pkg.packed_bwd(q, k, v, o, do, lse[:2], cu), lambda: pkg.packed_fwd(q.transpose(1, 2), k, v, cu)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: pkg.packed_fwd(q, k.float(), v, cu), lambda: pkg.packed_fwd(q.double(), k.double(), v.double(), cu)):
        with pytest.raises(TypeError):
            bad()
    h = [t.half() for t in (q, k, v)]
    with pytest.raises(pkg.WaveHipError, match="fp16"):
        pkg.packed_bwd(*h, o.half(), do.half(), lse, cu)
    assert pkg.packed_fwd(q[:0], k[:0], v[:0], cu)[0].shape[0] == 0
    assert pkg.packed_fwd(q, k, v, cu[:1])[0].shape == q.shape  # no sequence: nothing written
