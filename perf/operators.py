"""Cases of the token-by-token serving operators: a 4-bit grouped Linear for few
rows, the append of keys and values to a paged cache with RoPE on the way, and
the attention of one new token per sequence over that cache.

`run` computes an operator either from elementary torch operations in float32,
rounded once at the end (`own` false), or by the package's entry points
(`own` true).  `exact` restates each operator in float64.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _ops():
    path = os.path.join(os.getcwd(), "esm-cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from esm_b200 import ops

    return ops


# ------------------------------------------------------------------- cases
def _linear(name, M, N, K, group, dtype, scale_dtype, zeros, bias):
    return dict(name=name, op="linear_w4", M=M, N=N, K=K, group=group, dtype=dtype,
                scale_dtype=scale_dtype, zeros=zeros, bias=bias)


def _append(name, B, new_lo, new_hi, ctx_hi, Hq, Hkv, dh, rot, page, dtype, cache_dtype):
    return dict(name=name, op="kv_append", B=B, new_lo=new_lo, new_hi=new_hi, ctx_hi=ctx_hi, Hq=Hq,
                Hkv=Hkv, dh=dh, rot=rot, page=page, dtype=dtype, cache_dtype=cache_dtype)


def _attend(name, B, lo, hi, empty, Hq, Hkv, dh, page, window, dtype):
    return dict(name=name, op="attention_decode", B=B, lo=lo, hi=hi, empty=empty, Hq=Hq, Hkv=Hkv,
                dh=dh, page=page, window=window, dtype=dtype)


def listed():
    return [
        # One token through a d x d projection of the 650M width in the package's own float32: the
        # smallest product of a step, all latency.
        _linear("w4_1x1280x1280_f32", 1, 1280, 1280, 128, "f32", "f32", False, True),
        # Four sequences through the feed-forward of the 3B width, finer groups.
        _linear("w4_4x10240x2560_f32_g64", 4, 10240, 2560, 64, "f32", "f32", False, True),
        # A decoding batch with zero points, 32-wide groups and sizes that fill no tile.
        _linear("w4_13x5121x4100_f16_g32z", 13, 5121, 4100, 32, "f16", "f16", True, True),
        # One token through a wide decoder's feed-forward: 117 MB of weights, all bandwidth.
        _linear("w4_1x28672x8192_bf16", 1, 28672, 8192, 128, "bf16", "bf16", False, False),
        # One new token of one sequence, 650M heads: latency.
        _append("append_1seq_1tok", 1, 1, 1, 300, 20, 20, 64, 64, 16, "f32", "f32"),
        # A decoding batch with grouped heads, one token each.
        _append("append_256seq_1tok_gqa", 256, 1, 1, 200, 32, 8, 128, 128, 16, "bf16", "bf16"),
        # A packed batch of protein-length prompts (90 to 250 residues), float32 activations into a
        # bfloat16 cache.
        _append("append_192seq_prompts", 192, 90, 250, 0, 20, 20, 64, 64, 16, "f32", "bf16"),
        # Two long prompts behind a cached prefix, half of each head rotated.
        _append("append_2seq_16k", 2, 16000, 16385, 100, 32, 8, 128, 64, 64, "bf16", "bf16"),
        # One protein-length sequence, 650M heads in float32: latency.
        _attend("attend_1seq_130_f32", 1, 130, 130, False, 20, 20, 64, 16, 0, "f32"),
        # A ragged float32 batch of the 650M heads, one sequence still empty.
        _attend("attend_48seq_1k_f32", 48, 122, 1026, True, 20, 20, 64, 16, 0, "f32"),
        # A ragged decoding batch with grouped heads.
        _attend("attend_64seq_4k_bf16_gqa", 64, 1, 4099, False, 32, 8, 128, 16, 0, "bf16"),
        # One long context: the split over the cache's length.
        _attend("attend_1seq_128k_bf16_gqa", 1, 131071, 131071, False, 32, 8, 128, 64, 0, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_w4", "kv_append", "attention_decode"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "linear_w4":
        M, N, K = _log_int(rng, 1, 16), _log_int(rng, 100, 28672), _log_int(rng, 100, 16384)
        while M * N * K > 28672 * 8192:  # at most the work of the largest listed product
            M, N, K = max(1, M // 2), max(100, N * 3 // 4), max(100, K * 3 // 4)
        if rng.random() < 0.7:  # mostly whole groups, as real layers have
            K = -(-K // 128) * 128 if K > 128 else 128
        return dict(op=op, M=M, N=N, K=K, group=rng.choice([32, 64, 128]), dtype=dtype,
                    scale_dtype=rng.choice([dtype, "f32"]), zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.5)
    Hkv = rng.choice([1, 2, 3, 4, 5, 8, 16, 20])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    while Hkv * group > 64:
        group = max(1, group // 2)
    dh = rng.choice([16, 24, 32, 64, 64, 96, 128, 128])
    page = rng.choice([1, 8, 16, 16, 20, 32, 64, 128])
    heads = (Hkv * group + 2 * Hkv) * dh
    if op == "kv_append":
        most = 32768 * 48 * 128 // heads  # tokens at the largest listed case's values
        T = _log_int(rng, 1, min(32768, most))
        B = _log_int(rng, 1, min(T, 256))
        hi = max(1, T // B)
        return dict(op=op, B=B, new_lo=max(1, hi // 2), new_hi=hi, ctx_hi=rng.choice([0, 17, 200]),
                    Hq=Hkv * group, Hkv=Hkv, dh=dh, rot=rng.choice([dh, dh, dh // 2 // 2 * 2]), page=page,
                    dtype=dtype, cache_dtype=rng.choice([dtype, "bf16" if dtype == "f32" else dtype]))
    most = 131072 * 8 * 128 * 2 // (Hkv * dh * _BYTES[dtype])  # keys at the largest listed case's bytes
    keys = _log_int(rng, 1, min(131072, most))
    B = _log_int(rng, 1, min(keys, 128))
    hi = max(1, keys // B)
    return dict(op=op, B=B, lo=rng.choice([1, max(1, hi // 2)]), hi=hi, empty=B > 2 and rng.random() < 0.3,
                Hq=Hkv * group, Hkv=Hkv, dh=dh, page=page, window=rng.choice([0, 0, 0, max(1, hi // 3)]),
                dtype=dtype)


def _lengths(n, lo, hi):
    """n lengths in [lo, hi]; the case alone sets them, so that work() knows them too."""
    r = random.Random("%d %d %d" % (n, lo, hi))
    return [r.randint(lo, hi) for _ in range(n)]


def _decode_lengths(case):
    lens = _lengths(case["B"], case["lo"], case["hi"])
    if case["empty"]:
        lens[1] = 0
    return lens


def _append_lengths(case):
    return (_lengths(case["B"], case["new_lo"], case["new_hi"]),
            _lengths(case["B"], 0, case["ctx_hi"]))


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear_w4":
        M, N, K, G = (case[k] for k in ("M", "N", "K", "group"))
        groups = -(-K // G)
        nbytes = (N * -(-K // 2) + N * groups * (_BYTES[case["scale_dtype"]] + (1 if case["zeros"] else 0))
                  + M * K * e + M * N * e + (4 * N if case["bias"] else 0))
        return {"bytes": nbytes, "flops": 2 * M * N * K}
    if case["op"] == "kv_append":
        new, ctx = _append_lengths(case)
        T, c = sum(new), _BYTES[case["cache_dtype"]]
        Hq, Hkv, dh, rot = (case[k] for k in ("Hq", "Hkv", "dh", "rot"))
        rows = max((n + x for n, x in zip(new, ctx)), default=0)  # table rows in use, cos and sin
        pages = sum(-(-(n + x) // case["page"]) for n, x in zip(new, ctx))
        nbytes = (T * (Hq + 2 * Hkv) * dh * (e + c) + min(T, rows) * rot * 4 + 4 * pages
                  + 4 * (2 * case["B"] + 1))
        return {"bytes": nbytes, "flops": 3 * T * (Hq + Hkv) * rot}
    lens = [min(n, case["window"]) if case["window"] else n for n in _decode_lengths(case)]
    Hq, Hkv, dh = case["Hq"], case["Hkv"], case["dh"]
    keys = sum(lens)
    nbytes = (2 * keys * Hkv * dh * e + 2 * case["B"] * Hq * dh * e + 4 * case["B"] * (Hq + 1)
              + 4 * sum(-(-n // case["page"]) for n in lens))
    return {"bytes": nbytes, "flops": 4 * keys * Hq * dh}


# ------------------------------------------------------------------ inputs
def _paged_cache(case, capacity, dtype, g, dev):
    """Pages for `capacity[b]` tokens of each sequence, in scattered order, with spare ones."""
    page = case["page"]
    need = [-(-n // page) for n in capacity]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(need), max(1, max(need))), dtype=torch.int32, device=dev)
    cols = torch.arange(table.shape[1], device=dev)
    need_t = torch.tensor(need, device=dev)
    first = torch.cumsum(need_t, 0) - need_t
    at = (first[:, None] + cols[None, :]).clamp(max=total - 1)
    table.copy_(torch.where(cols[None, :] < need_t[:, None], order[at], table))
    shape = (total, page, case["Hkv"], case["dh"])
    k = torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)
    v = torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)
    return k, v, table


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "linear_w4":
        M, N, K, G = (case[k] for k in ("M", "N", "K", "group"))
        groups = -(-K // G)
        s = dict(case)
        s["x"] = torch.randn((M, K), generator=g, device=dev).to(dtype)
        s["wq"] = torch.randint(0, 256, (N, -(-K // 2)), generator=g, device=dev, dtype=torch.uint8)
        s["scales"] = (0.002 + 0.006 * torch.rand((N, groups), generator=g, device=dev)).to(
            _DTYPES[case["scale_dtype"]])
        s["z"] = (torch.randint(0, 16, (N, groups), generator=g, device=dev, dtype=torch.uint8)
                  if case["zeros"] else None)
        s["b"] = torch.randn((N,), generator=g, device=dev) * 0.02 if case["bias"] else None
        return s
    s = dict(case)
    Hq, Hkv, dh = case["Hq"], case["Hkv"], case["dh"]
    if case["op"] == "kv_append":
        new, ctx = _append_lengths(case)
        s["k_cache"], s["v_cache"], s["table"] = _paged_cache(
            case, [n + x for n, x in zip(new, ctx)], _DTYPES[case["cache_dtype"]], g, dev)
        T = sum(new)
        s["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
        s["ctx"] = torch.tensor(ctx, device=dev, dtype=torch.int32)
        # The projections' output, heads of q, k and v side by side in each token's row.
        qkv = torch.randn((T, Hq + 2 * Hkv, dh), generator=g, device=dev).to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        rows = max(n + x for n, x in zip(new, ctx))
        half = case["rot"] // 2
        inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * inv[None, :]
        s["cos"] = torch.cat([angle.cos(), angle.cos()], 1).float()
        s["sin"] = torch.cat([angle.sin(), angle.sin()], 1).float()
        return s
    lens = _decode_lengths(case)
    s["k_cache"], s["v_cache"], s["table"] = _paged_cache(case, lens, dtype, g, dev)
    s["lens"] = torch.tensor(lens, device=dev, dtype=torch.int32)
    s["q"] = torch.randn((case["B"], Hq, dh), generator=g, device=dev).to(dtype)
    return s


# -------------------------------------------------------------- plain forms
def _plain_linear_w4(s):
    N, K, G = s["N"], s["K"], s["group"]
    q = torch.stack([s["wq"] & 15, s["wq"] >> 4], dim=-1).reshape(N, -1)[:, :K].float()
    z = 8.0 if s["z"] is None else s["z"].float().repeat_interleave(G, 1)[:, :K]
    w = (q - z) * s["scales"].float().repeat_interleave(G, 1)[:, :K]
    y = s["x"].float() @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(s["x"].dtype)


def _token_places(s):
    """Sequence and cache position of each packed token."""
    cu = s["cu"].long()
    T = s["k"].shape[0]
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, s["ctx"].long()[b] + t - cu[b]


def _plain_kv_append(s):
    b, pos = _token_places(s)
    page = s["table"][b, pos // s["page"]].long()
    slot = pos % s["page"]
    rot, half = s["rot"], s["rot"] // 2
    c, sn = s["cos"][pos][:, None, :half], s["sin"][pos][:, None, :half]

    def rotate(x):
        x = x.float()
        lo, hi = x[..., :half], x[..., half:rot]
        return torch.cat([lo * c - hi * sn, hi * c + lo * sn, x[..., rot:]], -1).to(s["k_cache"].dtype)

    s["k_cache"][page, slot] = rotate(s["k"])
    s["v_cache"][page, slot] = s["v"].to(s["v_cache"].dtype)
    return rotate(s["q"]), s["k_cache"], s["v_cache"]


def _plain_attention_decode(s):
    B, Hq, Hkv, dh = s["B"], s["Hq"], s["Hkv"], s["dh"]
    table = s["table"].long()
    k = s["k_cache"][table].reshape(B, -1, Hkv, dh).float()
    v = s["v_cache"][table].reshape(B, -1, Hkv, dh).float()
    q = s["q"].float().reshape(B, Hkv, Hq // Hkv, dh) * dh ** -0.5
    t = torch.arange(k.shape[1], device=k.device)[None, :]
    n = s["lens"].long()[:, None]
    seen = (t < n) & ((t >= n - s["window"]) if s["window"] else (t >= 0))
    sc = torch.matmul(q, k.permute(0, 2, 3, 1))
    sc = torch.where(seen[:, None, None, :], sc, torch.full_like(sc, -math.inf))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, :, None, None], v, torch.zeros_like(v))
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, torch.ones_like(total), total)
    return o.reshape(B, Hq, dh).to(s["q"].dtype), (top + torch.log(total)).reshape(B, Hq)


def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "linear_w4":
            return ops.linear_w4(s["x"], s["wq"], s["scales"], s["z"], s["b"], group_size=s["group"])
        if s["op"] == "kv_append":
            q = ops.kv_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"],
                                    s["ctx"], q=s["q"], cos=s["cos"], sin=s["sin"])
            return q, s["k_cache"], s["v_cache"]
        return ops.attention_decode_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                          scale=s["dh"] ** -0.5, window=s["window"], return_lse=True)
    if s["op"] == "linear_w4":
        return _plain_linear_w4(s)
    if s["op"] == "kv_append":
        return _plain_kv_append(s)
    return _plain_attention_decode(s)


# --------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear_w4":
        N, K, G = case["N"], case["K"], case["group"]
        x = s["x"].double()
        cols = torch.arange(K, device=x.device)
        parts = []
        for n0 in range(0, N, 4096):  # rows of W in blocks, to bound the memory
            rows = slice(n0, min(N, n0 + 4096))
            byte = s["wq"][rows].int()[:, cols // 2]
            q = torch.bitwise_right_shift(byte, (4 * (cols % 2)).int()[None, :]) % 16
            zero = s["z"][rows].double()[:, cols // G] if case["zeros"] else 8.0
            w = s["scales"][rows].double()[:, cols // G] * (q.double() - zero)
            y = torch.einsum("mk,nk->mn", x, w)
            parts.append(y + s["b"][rows].double() if case["bias"] else y)
        return torch.cat(parts, 1)
    if case["op"] == "kv_append":
        new, ctx = _append_lengths(case)
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        cos, sin = s["cos"].double(), s["sin"].double()
        half, rot = case["rot"] // 2, case["rot"]
        q_out, at = [], 0

        def rotated(x, pos):
            z = x.double()
            if half:
                pair = torch.complex(z[..., :half].contiguous(), z[..., half:rot].contiguous())
                turn = torch.complex(cos[pos, :half], sin[pos, :half])[:, None, :]
                z[..., :rot] = torch.cat([(pair * turn).real, (pair * turn).imag], -1)
            return z

        for b, (n, x) in enumerate(zip(new, ctx)):
            pos = torch.arange(x, x + n, device=cos.device)
            where = (s["table"][b].long()[pos // case["page"]], pos % case["page"])
            k_cache[where] = rotated(s["k"][at:at + n].clone(), pos)
            v_cache[where] = s["v"][at:at + n].double()
            q_out.append(rotated(s["q"][at:at + n].clone(), pos))
            at += n
        return torch.cat(q_out), k_cache, v_cache
    B, Hq, Hkv, dh = case["B"], case["Hq"], case["Hkv"], case["dh"]
    out = torch.zeros((B, Hq, dh), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=out.device)
    for b, n in enumerate(_decode_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == first:
            continue
        t = torch.arange(first, n, device=out.device)
        where = (s["table"][b].long()[t // case["page"]], t % case["page"])
        k, v = s["k_cache"][where].double(), s["v_cache"][where].double()
        q = s["q"][b].double().reshape(Hkv, Hq // Hkv, dh)
        sc = torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(dh)
        out[b] = torch.einsum("hgt,thd->hgd", torch.softmax(sc, -1), v).reshape(Hq, dh)
        lse[b] = torch.logsumexp(sc, -1).reshape(Hq)
    return out, lse
