"""The token-by-token serving operators on the GPU against float64.

Tolerances count roundings.  With u = 2^-24 (half a float32 step) and e the
output type's half step (2^-24, 2^-11 or 2^-8):
  linear_w4   any order of summation is off by at most (longest chain of
              additions) * u of sum|x w|, twice that where the tensor cores
              truncate; the chains here are at most K/32 + 40 long.
  append      two products and their sum in float32: 2 u (|x c| + |y s|),
              then one rounding.
  attention   a score is off by (dh/16 + 16) 2u of sum|q k|, times scale; its
              exponential by that and 2^-21; sums of n terms by n u; the
              probabilities of 16-bit caches enter the tensor cores in two
              parts, off by 2^-16.  Twice, for the quotient.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _types():
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half_step(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half the spacing of the type's subnormal numbers."""
    import torch

    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def _gen(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ linear_w4
def _w4_case(cuda, M, N, K, group, dtype, sdtype, zeros, bias, seed=0, pad=0):
    import torch

    g = _gen(seed + M * 31 + N * 7 + K)
    groups = -(-K // group)
    x = torch.randn((M, K), generator=g, device=cuda).to(dtype)
    wq = torch.randint(0, 256, (N, (K + 1) // 2 + pad), generator=g, device=cuda, dtype=torch.uint8)[:, :(K + 1) // 2]
    s = (0.01 + torch.rand((N, groups), generator=g, device=cuda)).to(sdtype)
    z = torch.randint(0, 16, (N, groups), generator=g, device=cuda, dtype=torch.uint8) if zeros else None
    b = torch.randn((N,), generator=g, device=cuda) if bias else None
    return x, wq, s, z, b


def _w4_want(x, wq, s, z, b, group):
    import torch

    K = x.shape[1]
    q = torch.stack([wq & 15, wq >> 4], -1).flatten(1)[:, :K].double()
    zz = torch.full_like(s, 8, dtype=torch.float64) if z is None else z.double()
    w = (q - zz.repeat_interleave(group, 1)[:, :K]) * s.double().repeat_interleave(group, 1)[:, :K]
    y, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    return (y if b is None else y + b.double()), (mag if b is None else mag + b.double().abs())


def _w4_check(x, wq, s, z, b, group, out=None):
    from esm_b200 import ops

    got = ops.linear_w4(x, wq, s, z, b, group_size=group) if out is None else out
    ops.synchronize()
    want, mag = _w4_want(x, wq, s, z, b, group)
    K = x.shape[1]
    # mag uses |w|; the sums may run over q x before the zero point is taken
    # off, so count 16 s |x| as well.
    import torch

    big = 16 * (x.double().abs() @ s.double().repeat_interleave(group, 1)[:, :K].t())
    tol = (K / 32 + 40) * 2 * U * (mag + big) + _half_step(x.dtype) * want.abs() * (1 + 2.0**-6) + _tiny(x.dtype)
    assert got.dtype == x.dtype and got.shape == want.shape
    worst = ((got.double() - want).abs() / tol).max() if got.numel() else torch.zeros(())
    assert float(worst) <= 1.0, f"{float(worst):.3g} of the tolerance"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,group,zeros,bias", [
    (1, 1, 1, 128, False, True), (1, 16, 128, 128, False, False), (1, 17, 129, 32, True, True),
    (2, 40, 96, 32, True, False), (3, 65, 320, 64, False, True), (7, 33, 1000, 64, True, True),
    (8, 128, 4096, 128, False, False), (9, 129, 1025, 128, True, False), (16, 200, 512, 32, False, True),
    (33, 70, 640, 64, True, True), (65, 50, 256, 128, True, True), (130, 31, 384, 32, False, False),
    (1, 2561, 1280, 128, False, True), (4, 640, 10240, 64, True, False), (64, 40, 2100, 128, True, False),
    (1, 20, 131072, 128, False, False), (5, 33, 70000, 32, True, True), (16, 3000, 4096, 128, False, True),
    (2, 9000, 2048, 32, False, False), (20, 500, 16384, 64, True, True),
])
def test_linear_w4(cuda, M, N, K, group, zeros, bias, dtype):
    t = _types()
    _w4_check(*_w4_case(cuda, M, N, K, group, t[dtype], t[dtype], zeros, bias), group)


@pytest.mark.parametrize("dtype,sdtype", [("f32", "bf16"), ("f16", "f32"), ("bf16", "f16")])
def test_linear_w4_scale_types(cuda, dtype, sdtype):
    t = _types()
    _w4_check(*_w4_case(cuda, 5, 96, 640, 64, t[dtype], t[sdtype], True, True), 64)


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (3, 0), (16, 0), (0, 1), (0, 8)])
def test_linear_w4_layouts(cuda, pad, shift):
    """Row strides and bases that allow 16-byte reads, and ones that do not;
    strided x; neither the neighbours' bytes nor the bits behind an odd K are
    used."""
    import torch

    g = _gen(pad * 10 + shift)
    for K in (256, 255):
        cols = (K + 1) // 2
        M, N = 3, 50
        store = torch.randint(0, 256, (N * (cols + pad) + 32,), generator=g, device=cuda, dtype=torch.uint8)
        wq = store[shift:shift + N * (cols + pad)].view(N, cols + pad)[:, :cols]
        wide = torch.randn((M, 3 * K), generator=g, device=cuda)
        x = wide[:, K:2 * K]
        s = torch.rand((N, 2), generator=g, device=cuda)
        _w4_check(x, wq, s, None, None, 128)


def test_linear_w4_empty(cuda):
    import torch

    from esm_b200 import ops

    for M, N, K in [(0, 8, 64), (3, 0, 64), (3, 8, 0)]:
        x = torch.ones((M, K), device=cuda)
        b = torch.arange(N, device=cuda, dtype=torch.float32)
        y = ops.linear_w4(x, torch.zeros((N, K // 2), device=cuda, dtype=torch.uint8),
                          torch.zeros((N, -(-K // 128)), device=cuda), None, b)
        ops.synchronize()
        assert y.shape == (M, N)
        if K == 0:
            assert torch.equal(y, b.expand(M, N))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_linear_w4_extremes(cuda, dtype):
    """Rows do not touch one another (a NaN or infinite row stays alone), the
    largest finite inputs stay finite, tiny ones are not lost."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    N, K = 24, 256
    g = _gen(3)
    wq = torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8)
    s = torch.full((N, 2), 2.0**-12, device=cuda)
    x = torch.randn((6, K), generator=g, device=cuda).to(t)
    clean = ops.linear_w4(x, wq, s)
    y = x.clone()
    y[1, 5] = float("nan")
    y[3, 7] = float("inf")
    dirty = ops.linear_w4(y, wq, s)
    ops.synchronize()
    keep = [0, 2, 4, 5]
    assert torch.equal(clean[keep], dirty[keep])
    assert bool(dirty[1].isnan().all())
    assert not bool(dirty[3].isfinite().any())
    big = torch.zeros((1, K), device=cuda, dtype=t)
    big[0, 3] = torch.finfo(t).max
    _w4_check(big, wq, s, None, None, 128)
    small = (x.float() * (2.0**-12 if dtype == "f16" else 2.0**-100)).to(t)
    _w4_check(small, wq, torch.ones((N, 2), device=cuda), None, None, 128)


def test_linear_w4_from_prep(cuda):
    import torch

    from esm_b200 import ops, prep

    rng = np.random.default_rng(1)
    w = (rng.standard_normal((80, 300)) * 0.05).astype(np.float32)
    wq, s = prep.quantize_weight_w4(w, 64)
    x = torch.randn((2, 300), generator=_gen(2), device=cuda)
    y = ops.linear_w4(x, torch.from_numpy(wq).to(cuda), torch.from_numpy(s).to(cuda), group_size=64)
    ops.synchronize()
    exact = x.double().cpu().numpy() @ w.T.astype(np.float64)
    # each weight is off by half a step of its group at most
    bound = x.double().abs().cpu().numpy() @ (np.repeat(s, 64, 1)[:, :300].T * 0.5) * (1 + 1e-5) + 1e-5
    assert np.all(np.abs(y.double().cpu().numpy() - exact) <= bound)


# ---------------------------------------------------------------- paged cache
def _cache(cuda, B, capacity, page, Hkv, dh, dtype, g, layout="slot", spare=2, fill=None):
    """Pages in scattered order; entries of the table behind a sequence's pages
    hold an id outside the cache."""
    import torch

    need = [-(-n // page) for n in capacity]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device=cuda).to(torch.int32)
    table = torch.full((B, max(1, max(need, default=1)) + 1), 2**30, dtype=torch.int32, device=cuda)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    out = []
    for _ in range(2):
        if layout == "slot":
            c = torch.randn((total, page, Hkv, dh), generator=g, device=cuda).to(dtype)
        else:  # [page, head, slot, i]
            c = torch.randn((total, Hkv, page, dh), generator=g, device=cuda).to(dtype).transpose(1, 2)
        if fill is not None:
            c.fill_(fill)
        out.append(c)
    return out[0], out[1], table


def _slots(table, b, n, page):
    import torch

    t = torch.arange(n, device=table.device)
    return table[b].long()[t // page], t % page


def _rope(dh, rows, cuda):
    import torch

    from esm_b200 import ops

    c, s = ops.rope_build_tables(rows, dh)
    return torch.from_numpy(c).to(cuda), torch.from_numpy(s).to(cuda)


def _rotate64(x, cos, sin, pos):
    """(rotated, sum of the products' magnitudes) in float64."""
    import torch

    x = x.double()
    rot = cos.shape[1]
    h = rot // 2
    c, s = cos.double()[pos, :h][:, None], sin.double()[pos, :h][:, None]
    lo, hi = x[..., :h], x[..., h:rot]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., rot:]], -1)
    m = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs(), 0 * x[..., rot:]], -1)
    return y, m


def _near(got, want, mag):
    tol = 2 * U * mag * (1 + 2.0**-6) + _half_step(got.dtype) * want.abs() * (1 + 2.0**-6) + _tiny(got.dtype)
    if got.numel():
        worst = ((got.double() - want).abs() / tol).max()
        assert float(worst) <= 1.0, f"{float(worst):.3g} of the tolerance"


@pytest.mark.parametrize("types", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("new,ctx,Hq,Hkv,dh,rot,page,layout", [
    ([1], [0], 1, 1, 16, 16, 16, "slot"), ([1, 1, 1], [0, 15, 16], 4, 2, 64, 64, 16, "slot"),
    ([5, 0, 17, 1], [3, 9, 0, 31], 6, 3, 24, 24, 8, "head"), ([33], [1], 8, 1, 128, 64, 20, "slot"),
    ([4, 4], [2, 0], 3, 3, 40, 20, 1, "head"), ([9], [7], 2, 1, 10, 6, 3, "slot"), ([2], [0], 2, 2, 7, 0, 4, "slot"),
    ([700, 800], [0, 5], 4, 4, 32, 32, 64, "slot"), ([5000, 5001], [0, 0], 2, 1, 16, 8, 16, "head"),
])
def test_append(cuda, types, new, ctx, Hq, Hkv, dh, rot, page, layout):
    import torch

    from esm_b200 import ops

    tin, tc = (_types()[t] for t in types)
    g = _gen(sum(new) + dh)
    B, T = len(new), sum(new)
    kc, vc, table = _cache(cuda, B, [n + c for n, c in zip(new, ctx)], page, Hkv, dh, tc, g, layout)
    qkv = torch.randn((T + 2, Hq + 2 * Hkv, dh), generator=g, device=cuda).to(tin)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), device=cuda, dtype=torch.int32)
    lens = torch.tensor(ctx, device=cuda, dtype=torch.int32)
    cos, sin = _rope(rot, max(n + c for n, c in zip(new, ctx)), cuda) if rot else (None, None)
    k0, v0 = kc.clone(), vc.clone()
    out = ops.kv_append_paged(k, v, kc, vc, table, cu, lens, q=q, cos=cos, sin=sin)
    ops.synchronize()
    written = torch.zeros(kc.shape[:2], dtype=torch.bool, device=cuda)
    for b in range(B):
        t = torch.arange(int(cu[b]), int(cu[b + 1]), device=cuda)
        pos = t - int(cu[b]) + ctx[b]
        where = (table[b].long()[pos // page], pos % page)
        written[where] = True
        for x, y in ((k[t], kc[where]), (q[t], out[t])):
            _near(y, *(_rotate64(x, cos, sin, pos) if rot else (x.double(), 0 * x.double())))
        assert torch.equal(vc[where], v[t].to(tc))
    assert torch.equal(kc[~written], k0[~written]) and torch.equal(vc[~written], v0[~written])


def test_append_agrees_with_rope_apply_varlen(cuda):
    """float32 into a float32 cache: the facade's own rotation, bit for bit."""
    import torch

    from esm_b200 import ops

    lens, H, dh = [5, 1, 30], 3, 64
    T = sum(lens)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), device=cuda, dtype=torch.int32)
    x = torch.randn((T, H, dh), generator=_gen(5), device=cuda)
    cos, sin = _rope(dh, 32, cuda)
    kc, vc, table = _cache(cuda, 3, lens, 16, H, dh, torch.float32, _gen(6))
    q = ops.kv_append_paged(x, x, kc, vc, table, cu, torch.zeros(3, dtype=torch.int32, device=cuda), q=x,
                            cos=cos, sin=sin)
    want = ops.rope_apply_varlen(x.clone(), cos, sin, cu, H, dh)
    ops.synchronize()
    assert torch.equal(q, want)
    for b, n in enumerate(lens):
        assert torch.equal(kc[_slots(table, b, n, 16)], want[int(cu[b]):int(cu[b + 1])])


def test_append_without_queries_and_padding_rows(cuda):
    """No q; tokens behind the last sequence are left out; an empty batch."""
    import torch

    from esm_b200 import ops

    kc, vc, table = _cache(cuda, 2, [4, 4], 4, 2, 32, torch.bfloat16, _gen(1))
    k0, v0 = kc.clone(), vc.clone()
    k = torch.randn((6, 2, 32), generator=_gen(2), device=cuda).to(torch.bfloat16)
    cu = torch.tensor([1, 2, 3], device=cuda, dtype=torch.int32)  # tokens 0, 3, 4, 5 belong to no sequence
    lens = torch.tensor([0, 3], device=cuda, dtype=torch.int32)
    assert ops.kv_append_paged(k, k, kc, vc, table, cu, lens) is None
    ops.synchronize()
    p = table.long()
    k0[p[0, 0], 0], k0[p[1, 0], 3] = k[1], k[2]
    v0[p[0, 0], 0], v0[p[1, 0], 3] = k[1], k[2]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    ops.kv_append_paged(k[:0], k[:0], kc, vc, table, cu, lens)
    ops.kv_append_paged(k, k, kc, vc, table, cu[:1], lens[:0])
    ops.synchronize()
    assert torch.equal(kc, k0)


def test_append_most_rows(cuda):
    """2^31 - 1 rows (one element, repeated), of which the last two belong to a
    sequence."""
    import torch

    from esm_b200 import ops

    T = 2**31 - 1
    k = torch.full((1, 1, 1), 3.0, dtype=torch.float16, device=cuda).expand(T, 1, 1)
    kc, vc = torch.zeros((2, 1, 4, 1, 1), dtype=torch.float16, device=cuda)
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    ops.kv_append_paged(k, k, kc, vc, table, torch.tensor([T - 2, T], dtype=torch.int32, device=cuda),
                        torch.tensor([1], dtype=torch.int32, device=cuda))
    ops.synchronize()
    for c in (kc, vc):
        assert c.flatten().tolist() == [0.0, 3.0, 3.0, 0.0]


def test_append_reports_bad_places(cuda):
    """A page id outside the cache, a position behind the page table or the
    RoPE tables, a negative length: the token is left out, the others are
    written, and synchronize() says so once."""
    import torch

    from esm_b200 import _lib, ops

    cos, sin = _rope(32, 8, cuda)
    for kind in ("page", "negative page", "table", "rope", "length"):
        kc, vc, table = _cache(cuda, 2, [8, 8], 4, 1, 32, torch.float32, _gen(1), spare=4)
        lens = torch.tensor([3, 3], device=cuda, dtype=torch.int32)
        use = table[:, :2].contiguous() if kind == "table" else table
        if kind == "page":
            table[0, 0] = kc.shape[0]
        elif kind == "negative page":
            table[0, 0] = -1
        elif kind == "table":
            lens[0] = 8
        elif kind == "rope":
            table[0, 2] = 0
            lens[0] = 8
        else:
            lens[0] = -1
        k0 = kc.clone()
        k = torch.randn((2, 1, 32), generator=_gen(2), device=cuda)
        cu = torch.arange(3, device=cuda, dtype=torch.int32)
        ops.kv_append_paged(k, k, kc, vc, use, cu, lens, cos=cos, sin=sin)
        with pytest.raises(_lib.EsmCudaError) as e:
            ops.synchronize()
        assert e.value.code == 2
        ops.synchronize()  # reported once
        where = (int(table[1, 0]), 3)
        assert torch.equal(vc[where], k[1])
        k0[where] = kc[where]
        assert torch.equal(kc, k0)


# ------------------------------------------------------------------ attention
def _attend_want(q, kc, vc, table, lens, scale, window, page):
    """(out, lse, magnitude of the score error's base, sum p|v|) in float64."""
    import torch

    B, Hq, dh = q.shape
    Hkv = kc.shape[2]
    out = torch.zeros((B, Hq, dh), dtype=torch.float64, device=q.device)
    mag, lse = torch.zeros_like(out), torch.full((B, Hq), -np.inf, dtype=torch.float64, device=q.device)
    base = torch.zeros((B, Hq), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        p, s = _slots(table, b, n, page)
        k, v = kc[p[first:], s[first:]].double(), vc[p[first:], s[first:]].double()
        k, v = (x.repeat_interleave(Hq // Hkv, 1) for x in (k, v))
        sc = scale * torch.einsum("hd,thd->ht", q[b].double(), k)
        base[b] = (abs(scale) * torch.einsum("hd,thd->ht", q[b].double().abs(), k.abs())).amax(1)
        pr = torch.softmax(sc, 1)
        out[b], mag[b] = torch.einsum("ht,thd->hd", pr, v), torch.einsum("ht,thd->hd", pr, v.abs())
        lse[b] = torch.logsumexp(sc, 1)
    return out, lse, base, mag


def _attend_check(q, kc, vc, table, lens, scale, window, page, got=None):
    import torch

    from esm_b200 import ops

    out, lse = got or ops.attention_decode_paged(q, kc, vc, table, lens, scale=scale, window=window, return_lse=True)
    ops.synchronize()
    want, wl, base, mag = _attend_want(q, kc, vc, table, lens, scale, window, page)
    n = max(1, int(lens.max()) if lens.numel() else 1)
    dh = q.shape[2]
    e_s = base * (dh / 16 + 16) * 2 * U
    rel = 2 * e_s + 2.0**-21 + n * U
    rel16 = rel + (0.0 if q.dtype == torch.float32 else 2.0**-16)
    tol = 2 * rel16[..., None] * mag + _half_step(q.dtype) * want.abs() * (1 + 2.0**-6) + _tiny(q.dtype)
    assert out.dtype == q.dtype and out.shape == want.shape and lse.dtype == torch.float32
    if out.numel():
        worst = ((out.double() - want).abs() / tol).max()
        assert float(worst) <= 1.0, f"out: {float(worst):.3g} of the tolerance"
    empty = wl == -np.inf
    assert torch.equal(lse == -np.inf, empty) and bool((out[empty] == 0).all())
    ltol = rel + e_s + 2.0**-22 * (1 + wl.abs())
    bad = ((lse.double() - wl).abs() > ltol) & ~empty
    assert not bool(bad.any()), float(((lse.double() - wl).abs() / ltol)[~empty].max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hkv,dh,page,window,layout", [
    ([1], 1, 1, 16, 16, 0, "slot"), ([0], 2, 1, 64, 16, 0, "slot"), ([1, 0, 2, 15, 16, 17], 4, 2, 64, 16, 0, "slot"),
    ([63, 64, 65, 127, 129, 255], 8, 8, 32, 16, 0, "head"), ([100, 7], 20, 20, 64, 16, 0, "slot"),
    ([31, 130], 9, 3, 24, 8, 0, "slot"), ([333, 1, 48], 32, 4, 128, 64, 0, "head"), ([77], 16, 1, 96, 20, 0, "slot"),
    ([50, 200], 40, 2, 128, 1, 0, "slot"), ([260], 33, 1, 40, 5, 0, "slot"), ([90, 17], 12, 3, 256, 16, 0, "slot"),
    ([1000, 3, 400], 10, 2, 64, 32, 37, "slot"), ([64, 500], 4, 4, 8, 16, 1, "head"), ([5000], 8, 2, 128, 16, 0, "slot"),
    ([3000, 1, 0, 2999], 6, 6, 64, 128, 1500, "slot"), ([40] * 70, 4, 4, 16, 16, 0, "slot"),
    ([9, 700] * 20, 5, 1, 64, 16, 0, "head"),
])
def test_attention_decode(cuda, dtype, lens, Hq, Hkv, dh, page, window, layout):
    import torch

    t = _types()[dtype]
    g = _gen(sum(lens) + dh + Hq)
    kc, vc, table = _cache(cuda, len(lens), lens, page, Hkv, dh, t, g, layout)
    q = torch.randn((len(lens), Hq + 1, dh), generator=g, device=cuda).to(t)[:, 1:]
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    _attend_check(q, kc, vc, table, n, dh**-0.5, window, page)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_decode_sharp_scores(cuda, dtype):
    """Scores of some hundreds: one key takes nearly all, the running maximum
    moves late, and probabilities underflow."""
    import torch

    t = _types()[dtype]
    g = _gen(11)
    lens = [700, 90, 5]
    kc, vc, table = _cache(cuda, 3, lens, 16, 2, 64, t, g)
    kc[int(table[0, 43]), 5] *= 12  # a late dominant key
    q = (4 * torch.randn((3, 8, 64), generator=g, device=cuda)).to(t)
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    _attend_check(q, kc, vc, table, n, 0.7, 0, 16)
    _attend_check(q, kc, vc, table, n, -0.7, 0, 16)
    _attend_check(q, kc, vc, table, n, 0.0, 0, 16)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_attention_decode_never_sees_stale_slots(cuda, dtype, junk):
    """Slots behind a sequence's end, before its window and in pages of no
    sequence hold NaN or infinities; table entries behind the end hold ids
    outside the cache."""
    import torch

    from esm_b200 import ops

    t = _types()[dtype]
    g = _gen(4)
    lens, page, window = [1, 30, 129, 0, 256], 16, 40
    kc, vc, table = _cache(cuda, 5, lens, page, 2, 64, t, g)
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device=cuda)
    for b, n in enumerate(lens):
        p, s = _slots(table, b, n, page)
        seen[p[max(0, n - window):], s[max(0, n - window):]] = True
    q = torch.randn((5, 6, 64), generator=g, device=cuda).to(t)
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    clean = ops.attention_decode_paged(q, kc, vc, table, n, 0.125, window, True)
    kc[~seen] = junk
    vc[~seen] = junk
    dirty = ops.attention_decode_paged(q, kc, vc, table, n, 0.125, window, True)
    ops.synchronize()
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dh,Hq,Hkv,page", [(64, 5, 5, 16), (128, 16, 1, 12), (256, 8, 1, 16), (32, 34, 2, 64)])
def test_attention_decode_short_sequences_in_short_and_long_tables(cuda, dtype, dh, Hq, Hkv, page):
    """Short sequences take another way through the kernel when their page table
    has room for long ones: every number of tiles either way."""
    import torch

    t, lens = _types()[dtype], [0, 1, 15, 16, 17, 33, 47, 64, 65, 90, 128]
    kc, vc, table = _cache(cuda, len(lens), lens, page, Hkv, dh, t, _gen(13))
    q = torch.randn((len(lens), Hq, dh), generator=_gen(14), device=cuda).to(t)
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    long = torch.cat([table, torch.full((len(lens), 1000), -1, dtype=torch.int32, device=cuda)], 1)
    for window in (0, 1, 20):
        _attend_check(q, kc, vc, table, n, dh**-0.5, window, page)
        _attend_check(q, kc, vc, long, n, dh**-0.5, window, page)
    for b in (3, 10):  # few items
        _attend_check(q[b:b + 1], kc, vc, table[b:b + 1], n[b:b + 1], dh**-0.5, 0, page)
        _attend_check(q[b:b + 1], kc, vc, long[b:b + 1], n[b:b + 1], dh**-0.5, 0, page)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_decode_query_layouts(cuda, dtype):
    """Queries that start off 16-byte boundaries, inside wider rows, heads apart
    and one row for all sequences, and a window beyond 31 bits."""
    import torch

    from esm_b200 import ops

    t, lens = _types()[dtype], [33, 5, 70]
    kc, vc, table = _cache(cuda, 3, lens, 16, 2, 64, t, _gen(11))
    n = torch.tensor(lens, device=cuda, dtype=torch.int32)
    wide = torch.randn((3, 7, 67), generator=_gen(12), device=cuda).to(t)
    for q in (wide[:, :4, :64], wide[:, 1:5, 3:], wide[:, 1:, 1:65][:, ::3], wide[:1, :4, 2:66].expand(3, 4, 64),
              wide[:, :1, 1:65].expand(3, 4, 64)):
        want = ops.attention_decode_paged(q.contiguous(), kc, vc, table, n, 0.125, return_lse=True)
        got = ops.attention_decode_paged(q, kc, vc, table, n, 0.125, 2**40, True)
        ops.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_decode_nan_stays_in_its_row(cuda):
    import torch

    from esm_b200 import ops

    for t in _types().values():
        kc, vc, table = _cache(cuda, 3, [50, 60, 70], 16, 2, 64, t, _gen(7))
        q = torch.randn((3, 4, 64), generator=_gen(8), device=cuda).to(t)
        n = torch.tensor([50, 60, 70], device=cuda, dtype=torch.int32)
        clean = ops.attention_decode_paged(q, kc, vc, table, n, 0.125)
        q2 = q.clone()
        q2[1, 2, 3] = float("nan")
        dirty = ops.attention_decode_paged(q2, kc, vc, table, n, 0.125)
        ops.synchronize()
        assert bool(dirty[1, 2].isnan().all())
        dirty[1, 2] = clean[1, 2]
        assert torch.equal(clean, dirty)


def test_attention_decode_reports_bad_lengths_and_pages(cuda):
    """A length behind the page table is cut to it, a negative one is empty, a
    bad page's keys are not seen; synchronize() says so."""
    import torch

    from esm_b200 import _lib, ops

    for t in (torch.float32, torch.bfloat16):
        kc, vc, table = _cache(cuda, 3, [64, 64, 64], 16, 2, 64, t, _gen(9))
        table = table[:, :4].contiguous()
        q = torch.randn((3, 4, 64), generator=_gen(10), device=cuda).to(t)
        ok = torch.tensor([64, 0, 20], device=cuda, dtype=torch.int32)
        want = ops.attention_decode_paged(q, kc, vc, table, ok, 0.125, return_lse=True)
        ops.synchronize()
        got = ops.attention_decode_paged(q, kc, vc, table, torch.tensor([65, -3, 20], device=cuda, dtype=torch.int32),
                                         0.125, return_lse=True)
        with pytest.raises(_lib.EsmCudaError) as e:
            ops.synchronize()
        assert e.value.code == 2
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        short = table.clone()
        short[0, 3] = kc.shape[0]
        short[2, 1] = -7
        got = ops.attention_decode_paged(q, kc, vc, short, ok, 0.125, return_lse=True)
        with pytest.raises(_lib.EsmCudaError):
            ops.synchronize()
        _attend_check(q, kc, vc, table, torch.tensor([48, 0, 16], device=cuda, dtype=torch.int32), 0.125, 0, 16, got)


def test_attention_decode_agrees_with_attention_varlen(cuda):
    """The last query row of the facade's packed attention."""
    import torch

    from esm_b200 import ops

    lens, H, dh = [40, 200, 1], 4, 64
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), device=cuda, dtype=torch.int32)
    T = sum(lens)
    q, k, v = (torch.randn((T, H, dh), generator=_gen(i), device=cuda) for i in range(3))
    q *= dh**-0.5
    full = ops.attention_varlen(q, k, v, cu, H, dh)
    kc, vc, table = _cache(cuda, 3, lens, 16, H, dh, torch.float32, _gen(5))
    ops.kv_append_paged(k, v, kc, vc, table, cu, torch.zeros(3, dtype=torch.int32, device=cuda))
    last = (cu[1:] - 1).long()
    got = ops.attention_decode_paged(q[last], kc, vc, table, torch.tensor(lens, device=cuda, dtype=torch.int32))
    ops.synchronize()
    # FP32 class of the facade's tests
    assert float(((got - full[last]).abs() / (1 + full[last].abs())).max()) <= 1e-4


def test_attention_decode_longest_sequence(cuda):
    """2^31 - 1 keys on one page that the table repeats: a query of zeros gives
    the mean of V, small integers whose sums a warp holds exactly (2^27 / 1184
    tiles of 16 keys times 2^7 times at most 8: below 2^24 units of 2^7); the
    join adds at most 1184 pieces, rounding each time, then one rounding."""
    import torch

    from esm_b200 import ops

    n, size = 2**31 - 1, 1 << 20
    kc = torch.ones((1, size, 1, 8), dtype=torch.float16, device=cuda)
    vc = torch.arange(1, 9, dtype=torch.float16, device=cuda).expand(1, size, 1, 8).contiguous()
    table = torch.zeros((1, 2048), dtype=torch.int32, device=cuda)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    q = torch.zeros((1, 1, 8), dtype=torch.float16, device=cuda)
    out, lse = ops.attention_decode_paged(q, kc, vc, table, lens, return_lse=True)
    ops.synchronize()
    tol = 2 * 1184 * U + _half_step(torch.float16)
    assert float((out.double()[0, 0] / torch.arange(1, 9, device=cuda) - 1).abs().max()) <= tol
    assert abs(float(lse) - np.log(n)) <= tol + 4 * U * np.log(n)
    # Its last keys, of an own page.
    last = torch.randn((2, 1, size, 1, 8), generator=_gen(6), device=cuda).half()
    kc, vc = torch.cat([kc, last[0]]), torch.cat([vc, last[1]])
    table[0, 2047] = 1
    q = torch.randn((1, 1, 8), generator=_gen(7), device=cuda).half()
    got = ops.attention_decode_paged(q, kc, vc, table, lens, 0.3, 77, True)
    short = torch.tensor([size - 1], dtype=torch.int32, device=cuda)
    want = ops.attention_decode_paged(q, kc, vc, table[:, 2047:], short, 0.3, 77, True)
    ops.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_decode_empty_batch_and_shared_pages(cuda):
    """B = 0; two sequences that share their prefix pages."""
    import torch

    from esm_b200 import ops

    kc, vc, table = _cache(cuda, 2, [64, 64], 16, 2, 64, torch.float16, _gen(3))
    table[1, :2] = table[0, :2]
    q = torch.randn((2, 4, 64), generator=_gen(4), device=cuda).half()
    n = torch.tensor([50, 61], device=cuda, dtype=torch.int32)
    _attend_check(q, kc, vc, table, n, 0.125, 0, 16)
    out, lse = ops.attention_decode_paged(q[:0], kc, vc, table, n[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_cache_offsets_past_32_bits(cuda):
    """Element offsets of a 5 GB cache pass 2^31."""
    import torch

    from esm_b200 import ops

    pages, page, H, dh = 9600, 64, 32, 128  # 2.5e9 elements
    kc = torch.zeros((pages, page, H, dh), dtype=torch.bfloat16, device=cuda)
    vc = torch.zeros_like(kc)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=cuda)
    x = torch.randn((130, H, dh), generator=_gen(1), device=cuda).to(torch.bfloat16)
    y = torch.randn((130, H, dh), generator=_gen(2), device=cuda).to(torch.bfloat16)
    cu = torch.tensor([0, 130], dtype=torch.int32, device=cuda)
    ops.kv_append_paged(x, y, kc, vc, table, cu, torch.tensor([10], dtype=torch.int32, device=cuda))
    ops.synchronize()
    assert torch.equal(kc[pages - 1, 10:], x[:54]) and torch.equal(vc[pages - 2, :12], y[118:])
    q = torch.randn((1, H, dh), generator=_gen(3), device=cuda).to(torch.bfloat16)
    _attend_check(q, kc, vc, table, torch.tensor([140], dtype=torch.int32, device=cuda), 0.09, 0, page)
    del kc, vc
    torch.cuda.empty_cache()


# ------------------------------------------------------- as they are used
def _decoder(cuda, dtype, seed=0, B=5, H=4, Hkv=2, dh=64, page=16, steps=6):
    """A one-layer attention block's weights, cache and inputs."""
    import torch

    from esm_b200 import prep

    rng = np.random.default_rng(seed)
    d = H * dh

    def weight(n, k):
        wq, s = prep.quantize_weight_w4((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32), 64)
        return torch.from_numpy(wq).to(cuda), torch.from_numpy(s).to(cuda)

    g = _gen(seed)
    cap = 40 + steps
    kc, vc, table = _cache(cuda, B, [cap] * B, page, Hkv, dh, dtype, g)
    cos, sin = _rope(dh, cap, cuda)
    ctx = torch.tensor([0, 7, 16, 39, 1][:B], device=cuda, dtype=torch.int32)
    xs = torch.randn((steps, B, d), generator=g, device=cuda).to(dtype)
    return dict(qkv=weight((H + 2 * Hkv) * dh, d), out=weight(d, d), kc=kc, vc=vc, table=table, cos=cos, sin=sin,
                ctx=ctx, xs=xs, H=H, Hkv=Hkv, dh=dh, page=page, cu=torch.arange(B + 1, device=cuda, dtype=torch.int32))


def _step(m, x, ctx):
    from esm_b200 import ops

    H, Hkv, dh = m["H"], m["Hkv"], m["dh"]
    qkv = ops.linear_w4(x, *m["qkv"], group_size=64).view(-1, H + 2 * Hkv, dh)
    q = ops.kv_append_paged(qkv[:, H:H + Hkv], qkv[:, H + Hkv:], m["kc"], m["vc"], m["table"], m["cu"], ctx,
                            q=qkv[:, :H], cos=m["cos"], sin=m["sin"])
    o = ops.attention_decode_paged(q, m["kc"], m["vc"], m["table"], ctx + 1, scale=dh**-0.5)
    return ops.linear_w4(o.flatten(1), *m["out"], group_size=64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decoding_steps(cuda, dtype):
    """Linear, append, attention, Linear over several steps, against the same
    steps in float64 from the same cache contents.  Each step starts from the
    float64 run's view of the cache, so errors do not pile up over steps; a
    step's own error is a few roundings of the type (8 e, with values of
    order 1 and row sums of |w| of order 16) plus float32 noise."""
    import torch

    t = _types()[dtype]
    m = _decoder(cuda, t)
    H, Hkv, dh, page = m["H"], m["Hkv"], m["dh"], m["page"]
    ctx = m["ctx"].clone()
    for x in m["xs"]:
        kc, vc = m["kc"].double(), m["vc"].double()
        y = _step(m, x, ctx)
        qkv, _ = _w4_want(x, *m["qkv"], None, None, 64)
        qkv = qkv.view(-1, H + 2 * Hkv, dh)
        pos = ctx.long()
        q, _ = _rotate64(qkv[:, :H], m["cos"], m["sin"], pos)
        k, _ = _rotate64(qkv[:, H:H + Hkv], m["cos"], m["sin"], pos)
        rows = torch.arange(len(pos), device=cuda)
        where = (m["table"].long()[rows, pos // page], pos % page)
        kc[where], vc[where] = k, qkv[:, H + Hkv:]
        o, _, _, _ = _attend_want(q, kc, vc, m["table"], ctx + 1, dh**-0.5, 0, page)
        want, mag = _w4_want(o.flatten(1), *m["out"], None, None, 64)
        e = _half_step(t)
        err = (y.double() - want).abs()
        # roundings on the way: qkv, rotated q and k (scores of order 1, each
        # off by about sum|q k| scale * 3 e <= 24 e), out, y.
        tol = (60 * e + 2.0**-18) * (mag + want.abs())
        assert float((err / tol).max()) <= 1.0
        assert float(err.norm() / want.norm()) <= 8 * e + 1e-6
        ctx += 1


def test_captured_steps_replay(cuda):
    """A captured step, replayed with new inputs and lengths, gives the eager
    calls' bits; two captured graphs replayed at once on two streams keep apart."""
    import torch

    from esm_b200 import ops

    models = [_decoder(cuda, torch.bfloat16, seed=s, steps=4) for s in (1, 2)]
    graphs = []
    for m in models:
        m["x_in"], m["ctx_in"] = m["xs"][0].clone(), m["ctx"].clone()
        m["eager"] = []
        kc, vc = m["kc"].clone(), m["vc"].clone()
        for i, x in enumerate(m["xs"]):
            m["eager"].append(_step(m, x, m["ctx"] + i).clone())
        m["kc"].copy_(kc)
        m["vc"].copy_(vc)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m["y"] = _step(m, m["x_in"], m["ctx_in"])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in models]
    for i in range(4):
        for m, g, s in zip(models, graphs, streams):
            with torch.cuda.stream(s):
                m["x_in"].copy_(m["xs"][i])
                m["ctx_in"].copy_(m["ctx"] + i) if i else m["ctx_in"].copy_(m["ctx"])
                for _ in range(3):  # appending again writes the same slots
                    g.replay()
        torch.cuda.synchronize()
        for m in models:
            assert torch.equal(m["y"], m["eager"][i])
    ops.synchronize()


def test_calls_from_two_threads_on_their_own_streams(cuda):
    import threading

    import torch

    models = [_decoder(cuda, torch.float32, seed=s) for s in (3, 4)]
    want = []
    for m in models:
        kc, vc = m["kc"].clone(), m["vc"].clone()
        want.append([_step(m, x, m["ctx"] + i).clone() for i, x in enumerate(m["xs"])])
        m["kc"].copy_(kc)
        m["vc"].copy_(vc)
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        m = models[i]
        with torch.cuda.stream(torch.cuda.Stream()) as _:
            s = torch.cuda.current_stream()
            got[i] = [_step(m, x, m["ctx"] + j) for j, x in enumerate(m["xs"])]
            s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_attention_decode_is_reproducible(cuda):
    import torch

    from esm_b200 import ops

    for t in _types().values():
        lens = [4000, 9, 2500]
        kc, vc, table = _cache(cuda, 3, lens, 16, 2, 64, t, _gen(3))
        q = torch.randn((3, 8, 64), generator=_gen(4), device=cuda).to(t)
        n = torch.tensor(lens, device=cuda, dtype=torch.int32)
        a = ops.attention_decode_paged(q, kc, vc, table, n, 0.125)
        for _ in range(5):
            assert torch.equal(a, ops.attention_decode_paged(q, kc, vc, table, n, 0.125))


def test_serving_refuses_wrong_tensors(cuda):
    import torch

    from esm_b200 import _lib, ops

    x = torch.zeros((2, 64), device=cuda)
    wq, s = torch.zeros((8, 32), dtype=torch.uint8, device=cuda), torch.zeros((8, 1), device=cuda)
    for args, kw in [((x.double(), wq, s), {}), ((x, wq.char(), s), {}), ((x, wq[:, :31], s), {}), ((x, wq, s[:, :0]), {}),
                     ((x, wq, s), dict(group_size=16)), ((x, wq.cpu(), s), {}), ((x.t(), wq, s), {}),
                     ((x, wq, s, wq[:, :1].int()), {}), ((x, wq, s, None, s[:, 0].half()), {}),
                     ((x, wq, s.int()), {})]:
        with pytest.raises(ValueError):
            ops.linear_w4(*args, **kw)
    kc, vc, table = _cache(cuda, 2, [16, 16], 16, 2, 64, torch.bfloat16, _gen(1))
    lens = torch.ones(2, dtype=torch.int32, device=cuda)
    cu = torch.arange(3, dtype=torch.int32, device=cuda)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=cuda)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=cuda)
    for bad in [dict(seq_lens=lens.long()), dict(q=q.half()), dict(page_table=table.long()), dict(page_table=table[:1]),
                dict(q=q[..., :32]), dict(seq_lens=lens[:1]), dict(v_cache=vc.half())]:
        a = dict(q=q, k_cache=kc, v_cache=vc, page_table=table, seq_lens=lens)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.attention_decode_paged(**a)
    with pytest.raises(_lib.EsmCudaError):  # 3 query heads over 2
        ops.attention_decode_paged(q[:, :3], kc, vc, table, lens)
    with pytest.raises(_lib.EsmCudaError):
        ops.attention_decode_paged(q, kc, vc, table, lens, window=-1)
    odd = torch.zeros((2, 16, 2, 68), dtype=torch.bfloat16, device=cuda)[..., :64]
    with pytest.raises(_lib.EsmCudaError):  # rows off 16-byte boundaries
        ops.attention_decode_paged(q, odd, odd.clone(), table, lens)
    for bad in [dict(k=k.half()), dict(v=k.float()), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:2]),
                dict(q=q[:1]), dict(cos=torch.zeros((4, 64), device=cuda)), dict(k=k[:, :1], v=k[:, :1])]:
        a = dict(k=k, v=k, k_cache=kc, v_cache=vc, page_table=table, cu_seqlens=cu, cache_lens=lens, q=q)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.kv_append_paged(**a)
    ops.synchronize()
