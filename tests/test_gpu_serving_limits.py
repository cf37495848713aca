"""The serving operators on the GPU at the ends of their ranges: the longest K of
every type, scores and sums that float32 holds only just, infinities, and calls
that are captured, overlap or want gradients.  Values of the operators in float64
and the meaning of U are those of test_gpu_serving."""
import os
import subprocess
import sys
import textwrap
from pathlib import Path

import numpy as np
import pytest

from test_gpu_serving import U, _attend_want, _cache, _gen, _half_step, _tiny, _types, _w4_case, _w4_check, _w4_want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,pad", [(1, 0), (1, 1), (3, 0), (3, 1)])
def test_linear_w4_longest_k(cuda, dtype, group, M, pad):
    """K = 131072 in every type and group, rows of wq on and off 16-byte
    boundaries."""
    t = _types()[dtype]
    _w4_check(*_w4_case(cuda, M, 33, 131072, group, t, t, True, True, pad=pad), group)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,group,zeros", [(1, 40, 256, 32, True), (3, 100, 1000, 64, False), (13, 50, 4100, 32, True),
                                               (20, 24, 640, 128, True), (2, 9000, 2048, 128, False)])
def test_linear_w4_infinite_inputs(cuda, dtype, M, N, K, group, zeros):
    """An infinite activation gives what its definition gives: an infinity of the
    weight's sign, NaN where the weight is 0 or two infinities meet; other rows
    are not touched."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    x, wq, s, z, b = _w4_case(cuda, M, N, K, group, t, t, zeros, True)
    clean = ops.linear_w4(x, wq, s, z, b, group_size=group)
    y = x.clone()
    y[0, K - 1] = float("inf")
    if M > 2:
        y[1, 5], y[1, 200] = float("-inf"), float("inf")
        y[2, 0] = float("-inf")
    got = ops.linear_w4(y, wq, s, z, b, group_size=group)
    ops.synchronize()
    rows = [0, 1, 2] if M > 2 else [0]
    want, _ = _w4_want(y[rows], wq, s, z, b, group)
    assert torch.equal(got[rows].isnan(), want.isnan())
    assert bool(want[0].isinf().any()) and torch.equal(got[rows].isposinf(), want.isposinf())
    assert torch.equal(got[rows].isneginf(), want.isneginf())
    rest = list(range(len(rows), M))
    assert torch.equal(got[rest], clean[rest])


def test_linear_w4_scales_near_the_largest(cuda):
    """Scales whose 2^24-fold is no float32 number, with sums that are."""
    import torch

    N, K = 40, 320
    x, wq, s, z, b = _w4_case(cuda, 3, N, K, 64, torch.float32, torch.float32, True, True)
    _w4_check(x, wq, s * 2.0**110, z, b, 64)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,size", [(1, 2000.0), (4, -60000.0)])
def test_linear_w4_outlier_column(cuda, dtype, M, size):
    """One activation far above the others, in a column whose weights are 0 in
    some rows: the zero point is taken off behind the sum, so such a row's bound
    counts the group's largest weight instead of its own (16 s |x|).  (60000 times
    a weight of 8 is beyond float16: there the definition's value rounds to an
    infinity.)"""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    x, wq, s, z, b = _w4_case(cuda, M, 64, 2048, 128, t, t, False, False)
    x[:, 700] = size
    wq[::2, 350] = (wq[::2, 350] & 0xF0) | 8
    got = ops.linear_w4(x, wq, s, z, b, group_size=128)
    ops.synchronize()
    want, mag = _w4_want(x, wq, s, z, b, 128)
    big = 16 * (x.double().abs() @ s.double().repeat_interleave(128, 1).t())
    tol = (2048 / 32 + 40) * 2 * U * (mag + big) + _half_step(t) * want.abs() * (1 + 2.0**-6) + _tiny(t)
    top = torch.finfo(t).max
    over = want.abs() > top + tol  # beyond every value that rounds to a finite one
    near = (want.abs() > top - tol) & ~over
    assert torch.equal(got.isinf() & ~near, over) and bool((got[over].sign() == want[over].sign()).all())
    fine = ~over & ~near
    assert bool(((got.double() - want).abs() <= tol)[fine].all()) and bool(fine[:, ::2].all())


@pytest.mark.parametrize("M,N,K,group,zeros", [(1, 64, 2048, 128, False), (4, 100, 1000, 32, True), (20, 40, 2048, 64, True),
                                               (2, 9000, 2048, 128, False)])
@pytest.mark.parametrize("size", [100.0, 2000.0, -60000.0, 2.0**30])
def test_linear_w4_float32_outlier_costs_others_nothing(cuda, M, N, K, group, zeros, size):
    """float32: an activation far above the others takes no bits from the rest of
    its row.  x enters within 2^-35 of the largest of its 256 columns; the groups'
    sums are exact; what follows (scales, groups, steps, shares: one chain of at
    most 2 K / group + 40 operations) rounds sums of |x w|."""
    import torch

    from esm_b200 import ops

    x, wq, s, z, b = _w4_case(cuda, M, N, K, group, torch.float32, torch.float32, zeros, False)
    col = 700
    x[:, col] = size
    zero = (z[:, col // group] if zeros else torch.full((N,), 8, device=cuda)).to(torch.uint8)
    wq[::2, col // 2] = (wq[::2, col // 2] & 0xF0) | zero[::2]
    got = ops.linear_w4(x, wq, s, z, b, group_size=group)
    ops.synchronize()
    want, mag = _w4_want(x, wq, s, z, b, group)
    q = torch.stack([wq & 15, wq >> 4], -1).flatten(1)[:, :K].double()
    w = (q - (8.0 if z is None else z.double().repeat_interleave(group, 1)[:, :K])) * s.double().repeat_interleave(group, 1)[:, :K]
    lost = torch.zeros_like(mag)
    for k in range(0, K, 256):
        lost += 2.0**-35 * x[:, k:k + 256].double().abs().amax(1)[:, None] * w[:, k:k + 256].abs().sum(1)[None, :]
    tol = (2 * K / group + 40) * U * mag + lost + U * want.abs()
    worst = float(((got.double() - want).abs() / tol).max())
    assert worst <= 1.0, worst


def _tables(table, long):
    """The page table as it is, or with room for far longer sequences (its other
    entries are outside the cache)."""
    import torch

    if not long:
        return table
    more = torch.full((table.shape[0], 1000), -1, dtype=torch.int32, device=table.device)
    return torch.cat([table, more], 1)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [2.0**25, 2.0**26, 2.0**27, -2.0**26])
def test_attention_decode_large_scores(cuda, dtype, top, long):
    """Scores (in powers of two) of about 2^25 to 2^27 that climb by 8 from tile to
    tile: products and scores are exact, so the probabilities are powers of 2^8,
    whatever the spacing of numbers as large as the scores."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    dh, tiles = 16, 5
    scale = np.float32(np.log(2.0))
    assert scale * np.float32(1.4426950408889634) == 1.0  # scores arrive as powers of two
    g = _gen(1)
    kc, vc, table = _cache(cuda, 1, [16 * tiles], 16, 1, dh, t, g)
    kc.zero_()
    q = torch.zeros((1, 2, dh), device=cuda, dtype=t)
    q[0, :, 0], q[0, :, 1] = 4096.0, 1.0
    step = 8.0 if abs(top) < 2.0**27 else 16.0
    for i in range(tiles):
        page = int(table[0, i])
        kc[page, :, :, 0] = top / 4096.0
        kc[page, :, :, 1] = step * (i + 8)
    n = torch.tensor([16 * tiles], device=cuda, dtype=torch.int32)
    out, lse = ops.attention_decode_paged(q, kc, vc, _tables(table, long), n, scale=float(scale), return_lse=True)
    ops.synchronize()
    v = torch.stack([vc[int(table[0, i]), :, 0] for i in range(tiles)]).double()  # [tiles, 16, dh]
    p = 2.0 ** (step * torch.arange(1 - tiles, 1, device=cuda, dtype=torch.float64))
    p /= 16 * p.sum()
    want, mag = torch.einsum("i,ijd->d", p, v), torch.einsum("i,ijd->d", p, v.abs())
    # sums of 80 terms, exponentials 2^-21, two 16-bit parts 2^-16; the tensor cores' truncation twice
    tol = 2 * (2.0**-21 + 80 * 2 * U + (0.0 if dtype == "f32" else 2.0**-16)) * mag + _half_step(t) * want.abs() * (1 + 2.0**-6)
    assert bool(((out[0].double() - want).abs() <= tol + _tiny(t)).all())
    top_score = (top + step * (tiles + 7)) * np.log(2.0)
    assert float((lse.double() - top_score - np.log(16.0)).abs().max()) <= 4 * U * abs(top_score) + 1e-2


def test_attention_decode_long_sums_of_one_sign(cuda):
    """2^31 - 1 keys of equal weight and values in [1, 2): sums that lost a little
    at every step would be off by far more than the output's rounding.  A warp
    adds up at most 2^27 / 1184 + 1 tiles, each addition rounded to nearest by at
    most U of a sum that grows evenly: roundings of a random sign pile up to
    sqrt(tiles / 3) U, of which 16 times is allowed, beside half a step of the
    output and a few roundings of the join."""
    import torch

    from esm_b200 import ops

    n, size, dh = 2**31 - 1, 1 << 20, 8
    kc = torch.zeros((1, size, 1, dh), dtype=torch.float16, device=cuda)
    vc = (1.0 + torch.rand((1, size, 1, dh), generator=_gen(2), device=cuda)).half()
    table = torch.zeros((1, 2048), dtype=torch.int32, device=cuda)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    q = torch.zeros((1, 1, dh), dtype=torch.float16, device=cuda)
    out = ops.attention_decode_paged(q, kc, vc, table, lens)
    ops.synchronize()
    want = (2048 * vc.double().sum(1)[0, 0] - vc[0, -1, 0].double()) / n
    tol = _half_step(torch.float16) * (1 + 2.0**-6) + (16 * np.sqrt((2**27 / 1184 + 1) / 3) + 2 * 1184**0.5 * 16) * U
    worst = float(((out.double()[0, 0] - want) / want).abs().max())
    assert worst <= tol, (worst, tol)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dh,Hq,Hkv,page", [(64, 4, 2, 16), (128, 12, 1, 16), (24, 3, 3, 12), (256, 2, 2, 16)])
def test_attention_decode_infinite_keys(cuda, dtype, dh, Hq, Hkv, page, long):
    """An infinite element of a seen key: its score is minus infinity, a probability
    of 0, for the heads whose query is negative there, and plus infinity, NaN by
    the definition, for the others; the heads of another K are not touched."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    lens = [1, 50, 130]
    g = _gen(dh + Hq)
    kc, vc, table = _cache(cuda, 3, lens, page, Hkv, dh, t, g)
    q = torch.randn((3, Hq, dh), generator=g, device=cuda).to(t)
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    table = _tables(table, long)
    d = dh - 3
    assert bool((q[:, :, d] != 0).all())
    clean = ops.attention_decode_paged(q, kc, vc, table, n, dh**-0.5, return_lse=True)
    for b, at in ((1, 0), (1, 33), (2, 129)):
        kc[int(table[b, at // page]), at % page, 0, d] = float("inf")
    got = ops.attention_decode_paged(q, kc, vc, table, n, dh**-0.5, return_lse=True)
    ops.synchronize()
    group = Hq // Hkv
    drop = kc.clone()  # the same without those keys: a score that takes no part
    for b in (1, 2):
        gone = [0, 33] if b == 1 else [129]
        keep = torch.tensor([i for i in range(lens[b]) if i not in gone], device=cuda)
        pg, sl = table[b].long()[keep // page], keep % page
        k, v = kc[pg, sl, 0].double(), vc[pg, sl, 0].double()
        for h in range(group):
            if float(q[b, h, d]) > 0:
                assert bool(got[0][b, h].isnan().all()), (b, h)
                continue
            sc = dh**-0.5 * (k @ q[b, h].double())
            base = dh**-0.5 * float((k.abs() @ q[b, h].double().abs()).max())
            p = torch.softmax(sc, 0)
            want, mag = p @ v, p @ v.abs()
            e_s = base * (dh / 16 + 16) * 2 * U
            rel = 2 * e_s + 2.0**-21 + 200 * U + (0.0 if dtype == "f32" else 2.0**-16)
            tol = 2 * rel * mag + _half_step(t) * want.abs() * (1 + 2.0**-6) + _tiny(t)
            assert bool(((got[0][b, h].double() - want).abs() <= tol).all()), (b, h)
            assert abs(float(got[1][b, h]) - float(torch.logsumexp(sc, 0))) <= rel + e_s + 2.0**-21 * 10
    assert torch.equal(got[0][0], clean[0][0]) and torch.equal(got[0][:, group:], clean[0][:, group:])
    assert torch.equal(got[1][0], clean[1][0]) and torch.equal(got[1][:, group:], clean[1][:, group:])


@pytest.mark.parametrize("long", [False, True])
def test_attention_decode_largest_queries(cuda, long):
    """float32 queries that round up to infinity in fewer bits, keys so small that
    the scores are ordinary."""
    import torch

    from esm_b200 import ops

    g = _gen(5)
    lens, dh = [40, 7], 32
    kc, vc, table = _cache(cuda, 2, lens, 16, 1, dh, torch.float32, g)
    q = torch.randn((2, 3, dh), generator=g, device=cuda)
    big = torch.full((2, 3, dh), torch.finfo(torch.float32).max, device=cuda) * torch.sign(q)
    small = kc * 2.0**-126  # 2^128 q . 2^-126 k is of order 4 |k|
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    got = ops.attention_decode_paged(big, small, vc, _tables(table, long), n, 0.1, return_lse=True)
    ops.synchronize()
    want, wl, base, mag = _attend_want(big, small, vc, table, n, 0.1, 0, 16)
    # keys of 2^-126 times a normal number: those below it are subnormal, off by 2^-150 each (exactly held, but the
    # tensor cores may take subnormals for 0: up to 2^-126 of such an element, times 2^128 and 0.1)
    e_s = base * (dh / 16 + 16) * 2 * U
    rel = 2 * e_s[..., None] + 2.0**-21 + 40 * U
    tol = 2 * rel * mag + U * want.abs() * (1 + 2.0**-6)
    assert bool(((got[0].double() - want).abs() <= tol).all())
    assert bool(((got[1].double() - wl).abs() <= 2 * e_s + 2.0**-20).all())


def test_first_calls_of_a_process_inside_a_capture(cuda):
    """Nothing was called before the capture: the calls' contexts are opened inside
    it; the replayed graph gives the eager calls' bits."""
    code = """
        import torch
        from esm_b200 import ops
        dev = torch.device("cuda:0")
        g = torch.Generator(device=dev).manual_seed(1)
        x = torch.randn((40, 4096), generator=g, device=dev).bfloat16()
        wq = torch.randint(0, 256, (300, 2048), generator=g, dtype=torch.uint8, device=dev)
        s = torch.rand((300, 32), generator=g, device=dev)
        kc = torch.randn((8, 16, 2, 64), generator=g, device=dev).bfloat16()
        vc = torch.randn((8, 16, 2, 64), generator=g, device=dev).bfloat16()
        k = torch.randn((2, 2, 64), generator=g, device=dev).bfloat16()
        q = torch.randn((2, 4, 64), generator=g, device=dev).bfloat16()
        table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
        lens, cu = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([20, 50], [0, 1, 2]))
        after = lens + 1
        def step():
            ops.kv_append_paged(k, k, kc, vc, table, cu, lens)
            return (ops.linear_w4(x, wq, s), *ops.attention_decode_paged(q, kc, vc, table, after, 0.125, return_lse=True))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graph.replay()
        ops.synchronize()
        got = [y.clone() for y in got]
        for y, z in zip(got, step()):
            assert torch.equal(y, z)
        ops.synchronize()
        print("replayed")
    """
    root = Path(__file__).resolve().parents[1]
    env = dict(os.environ, PYTHONPATH=str(root / "esm-cpp_b200"))
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "replayed" in r.stdout, r.stderr[-2000:]


def test_a_bad_place_is_reported_from_any_stream(cuda):
    """One report for each time that somebody looks after a bad call, whichever
    stream it ran on, and none is lost."""
    import torch

    from esm_b200 import _lib, ops

    kc, vc, table = _cache(cuda, 1, [8], 4, 1, 32, torch.float32, _gen(1))
    k = torch.randn((1, 1, 32), generator=_gen(2), device=cuda)
    cu = torch.tensor([0, 1], device=cuda, dtype=torch.int32)
    bad = torch.tensor([-1], device=cuda, dtype=torch.int32)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(other):
            ops.kv_append_paged(k, k, kc, vc, table, cu, bad)
        other.synchronize()
        with pytest.raises(_lib.EsmCudaError) as e:
            ops.synchronize()
        assert e.value.code == 2
        ops.synchronize()


def test_appends_count_as_writes_for_autograd(cuda):
    import torch

    from esm_b200 import ops

    kc, vc, table = _cache(cuda, 1, [8], 4, 1, 32, torch.float32, _gen(1))
    k = torch.randn((1, 1, 32), generator=_gen(2), device=cuda)
    cu, lens = (torch.tensor(v, device=cuda, dtype=torch.int32) for v in ([0, 1], [2]))
    before = kc._version, vc._version
    ops.kv_append_paged(k, k, kc, vc, table, cu, lens)
    assert (kc._version, vc._version) == (before[0] + 1, before[1] + 1)
    w = torch.ones(1, device=cuda, requires_grad=True)
    y = (kc * w).sum()  # keeps kc for w's gradient
    ops.kv_append_paged(k, k, kc, vc, table, cu, lens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kc, vc = kc.clone(), vc.clone()  # inference tensors have no version
        ops.kv_append_paged(k, k, kc, vc, table, cu, lens)
    ops.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_prompts_causal_attention_row_by_row(cuda, dtype):
    """Causal attention within a prompt: one row of q per token, its sequence's page
    table, its position + 1 as the length."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    new, ctx, Hq, Hkv, dh, page = [5, 40, 1], [7, 0, 30], 4, 2, 64, 16
    g = _gen(8)
    T = sum(new)
    kc, vc, table = _cache(cuda, 3, [a + c for a, c in zip(new, ctx)], page, Hkv, dh, t, g)
    q = torch.randn((T, Hq, dh), generator=g, device=cuda).to(t)
    k = torch.randn((T, Hkv, dh), generator=g, device=cuda).to(t)
    v = torch.randn((T, Hkv, dh), generator=g, device=cuda).to(t)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), device=cuda, dtype=torch.int32)
    lens = torch.tensor(ctx, device=cuda, dtype=torch.int32)
    ops.kv_append_paged(k, v, kc, vc, table, cu, lens)
    b = torch.repeat_interleave(torch.arange(3, device=cuda), torch.tensor(new, device=cuda))
    seen = (lens[b] + torch.arange(T, device=cuda) - cu[b] + 1).int()
    out, lse = ops.attention_decode_paged(q, kc, vc, table[b], seen, dh**-0.5, return_lse=True)
    ops.synchronize()
    want, wl, base, mag = _attend_want(q, kc, vc, table[b], seen, dh**-0.5, 0, page)
    rel = 2 * base * (dh / 16 + 16) * 2 * U + 2.0**-21 + 50 * U + (0.0 if dtype == "f32" else 2.0**-16)
    tol = 2 * rel[..., None] * mag + _half_step(t) * want.abs() * (1 + 2.0**-6) + _tiny(t)
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_decode_of_scores_that_are_all_minus_infinity(cuda, dtype):
    """Nothing is left to attend to: zeros and minus infinity, as without keys."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    kc, vc, table = _cache(cuda, 2, [20, 40], 16, 1, 64, t, _gen(3))
    q = torch.randn((2, 2, 64), generator=_gen(4), device=cuda).to(t).abs()
    q[:, 1] *= -1
    kc[table[0, :2].long(), :, 0, 5] = float("-inf")
    n = torch.tensor([20, 40], device=cuda, dtype=torch.int32)
    for long in (False, True):
        out, lse = ops.attention_decode_paged(q, kc, vc, _tables(table, long), n, 0.125, return_lse=True)
        ops.synchronize()
        assert bool((out[0, 0] == 0).all()) and float(lse[0, 0]) == -np.inf
        assert bool(out[0, 1].isnan().all()) and bool(out[1].isfinite().all()) and bool(lse[1].isfinite().all())
