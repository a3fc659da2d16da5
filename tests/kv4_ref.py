"""The 4-bit cache and its attention in 64 bits, for the tests."""
import numpy as np
import torch

U = 2.0 ** -24
GROUP = 32


def f32(x):
    return x.to(torch.float32).to(torch.float64)


def quantise(x):
    """x [..., D] (16 bits) -> (codes, scale, minimum) [..., D] in 64 bits, a value's own group's; each operation of
    the definition rounded to f32, scale and minimum to f16."""
    D, codes, scales, minima = x.shape[-1], [], [], []
    x = x.to(torch.float64)
    for a in range(0, D, GROUP):
        v = x[..., a:a + GROUP]
        lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        s = f32(f32(hi - lo) / 15).to(torch.float16).to(torch.float64)
        m = lo.to(torch.float32).to(torch.float16).to(torch.float64)
        inv = torch.where(s > 0, f32(1 / s), torch.zeros_like(s))
        codes.append(f32(f32(v - m) * inv).round().clamp(0, 15))
        scales.append(s.expand_as(v))
        minima.append(m.expand_as(v))
    return torch.cat(codes, -1), torch.cat(scales, -1), torch.cat(minima, -1)


def stored(k, v):
    """(K values, V values, scale * code + |minimum| of K, scale * |code - 8| + |minimum + 8 scales| of V, scale * (code + 8) +
    |minimum + 8 scales| of V) that a cache of k, v [tokens][KVH][D] holds; values are NaN for a token and head that does not
    fit."""
    ok = ((k.double().abs() <= 32768) & (v.double().abs() <= 32768)).all(-1, keepdim=True)
    zero = torch.zeros((), dtype=k.dtype, device=k.device)
    (ck, sk, mk), (cv, sv, mv) = quantise(torch.where(ok, k, zero)), quantise(torch.where(ok, v, zero))
    nan = torch.full((), float("nan"), dtype=torch.float64, device=k.device)
    return torch.where(ok, mk + sk * ck, nan), torch.where(ok, mv + sv * cv, nan), mk.abs() + sk * ck, sv * (cv - 8).abs() + (mv + 8 * sv).abs(), sv * (cv + 8) + (mv + 8 * sv).abs()


def attention(q, kv, rows, lens, scale, causal):
    """(out, lse, tolerance of out before its rounding, of lse); q [rows][H][D], kv: stored() of each request's
    tokens; `rows` [(first, n)].

    A score is a sum over groups of scale * (a sum of products with codes) + minimum * (a sum of q), in f32: at most D + 16
    roundings, each within 2 U of the sum of magnitudes |q| (scale * code + |minimum|).  Where many rows come
    together a key is rounded to f16 (half a step relative, or half of the smallest step).  q is taken as f16 after a power
    of two has brought its row's largest value to 2^10 or above: exact, but for values below 2^-24 of
    that largest, off by 2^-35 of it.  The exponential adds 8 U and U for each unit of its argument.
    A weight p is rounded to f16 (half a step; below the normal range half of the smallest one, against a row's sum
    of at least one), and so are p * scale, whose rounding meets code - 8 (with the smallest step: up to 8), and minimum + 8 scales,
    or, where many rows come together, the value instead; sums over n keys, of p * scale * code, of 8 p * scale and of p * (minimum
    + 8 scales), add n U.  Numerator and denominator both carry the errors of
    the weights."""
    H, D = q.shape[1:]
    eps = 2.0 ** -10
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -np.inf, dtype=torch.float64, device=q.device)
    eo, el = torch.zeros_like(out), torch.zeros_like(lse)
    for (a, m), n, (k, v, mag, vc, parts) in zip(rows, lens, kv):
        if not m or not n:
            continue
        G = H // k.shape[1]
        k, v, mag, vc, parts = (t.repeat_interleave(G, dim=1) for t in (k, v, mag, vc, parts))
        qq = q[a:a + m].double()
        s = torch.einsum("qhd,khd->hqk", qq, k) * scale
        es = torch.einsum("qhd,khd->hqk", qq.abs(), mag * (2 * (D + 16) * U) + k.abs() * (eps / 2) + 2.0 ** -25) * scale
        es = es + torch.einsum("qh,khd->hqk", qq.abs().amax(-1), k.abs()) * (scale * 2.0 ** -35)
        if causal:
            hidden = torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + n - m
            s = s.masked_fill(hidden, -np.inf)
            es = es.masked_fill(hidden, 0.0)
            kv_seen = (~hidden).double()
        else:
            kv_seen = torch.ones((m, n), dtype=torch.float64, device=q.device)
        pr = torch.softmax(s, -1)
        bad = torch.isnan(pr)
        top = s.amax(-1, keepdim=True)
        ep = es + (8 + (s - top).abs().nan_to_num(posinf=0.0) * 2) * U
        # a value that no row of weight sees may be NaN
        vv = torch.where(torch.isnan(v), 0.0, v)
        rel = (pr * ep).sum(-1) + n * U
        o = torch.einsum("hqk,khd->qhd", pr, vv)
        w = torch.einsum("hqk,khd->qhd", pr * (ep + eps / 2 * (1 + eps)), vv.abs())
        w = w + torch.einsum("hqk,khd->qhd", pr, torch.maximum(vc, vv.abs()) * (eps / 2) + 2.0 ** -25) * (1 + eps)
        w = w + torch.einsum("hqk,khd->qhd", pr, vv.abs()) * (rel.t()[..., None] + 4 * U) + torch.einsum("hqk,khd->qhd", pr, parts) * (n * U)
        l = torch.exp(s - top).sum(-1)
        w = w + 2.0 ** -25 * torch.einsum("qk,khd->qhd", kv_seen, parts + 15) / l.t()[..., None]
        o[bad.any(-1).t()] = float("nan")
        out[a:a + m], eo[a:a + m] = o, w
        lse[a:a + m] = torch.logsumexp(s, -1).t()
        # the sum that the logarithm is of holds weights before their rounding
        el[a:a + m] = (rel + es.amax(-1) + 4 * U * (1 + lse[a:a + m].t().abs() + top[..., 0].abs())).t()
    return out, lse, eo, el
