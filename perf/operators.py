"""Workloads of the 8-bit product, the residual norm and cross attention.

Each case is one call that a serving or batch program makes: an 8-bit integer
product of a batch of tokens with a prepared weight, the norms around a block
with its gate and residual, and attention of ragged query rows to encoder
states.  `run` computes them in elementary torch operations, or, with `own`
set, through the library's entry points.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def needle():
    """The framework's package, imported by path (its folder is no identifier)."""
    if "needle_b200" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location("needle_b200", os.path.join(root, "needle-rs_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["needle_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["needle_b200"]


def code(name):
    n = needle()
    return {"f32": n.F32, "f16": n.F16, "bf16": n.BF16}[name]


def round_up(n, m):
    return (n + m - 1) // m * m


def int8_case(name, M, K, N, x, y, bias=False):
    return {"name": name, "op": "int8", "M": M, "K": K, "N": N, "x": x, "y": y, "bias": bias}


def norm_case(name, M, d, x, y, gate, sigmoid, post, scale, N=0):
    return {"name": name, "op": "norm", "M": M, "d": d, "x": x, "y": y, "gate": gate, "sigmoid": sigmoid, "post": post,
            "scale": scale, "N": N}


def attn_case(name, B, q_lo, q_hi, k_lo, k_hi, H, KVH, D, t, layout, keep=1.0, padded=False, lse=False, lens=1):
    return {"name": name, "op": "attn", "B": B, "q_lo": q_lo, "q_hi": q_hi, "k_lo": k_lo, "k_hi": k_hi, "H": H, "KVH": KVH,
            "D": D, "type": t, "layout": layout, "keep": keep, "padded": padded, "lse": lse, "lens": lens}


def listed():
    return [
        # one request's token through a projection of the shipped width: latency
        int8_case("int8_one_token", 1, 512, 2048, "f32", "f32"),
        # a decode step of 64 requests: the weight is what is read
        int8_case("int8_decode_64", 64, 4096, 4096, "bf16", "bf16"),
        # a batch of leftover tokens, no size a multiple of a tile, with a bias
        int8_case("int8_odd", 777, 1000, 1523, "f16", "f32", True),
        # a prefill chunk
        int8_case("int8_prefill", 8192, 4096, 4096, "bf16", "bf16"),
        # one token between two blocks of the shipped model (scalar sigmoid gate)
        norm_case("norm_one_token", 1, 512, "f32", "f32", "scalar", True, False, 1.0),
        # a decode batch with an f32 residual stream, both norms, and the 8-bit product that follows
        norm_case("norm_then_int8", 1001, 1000, "f32", "bf16", "channel", True, True, 1.0, 1536),
        # a prefill chunk with a gate for each token and channel
        norm_case("norm_prefill", 4096, 4096, "f32", "bf16", "token", True, True, 0.5),
        # the encoder's whole batch, 16-bit residual stream
        norm_case("norm_encoder_batch", 65536, 2048, "bf16", "bf16", "channel", False, True, 1.0),
        # one decode step of 256 requests over their prompts, head-major planes
        attn_case("attn_decode_256", 256, 1, 1, 64, 512, 8, 4, 64, "bf16", "head"),
        # few requests, long documents, padded keys masked out, the row statistics kept for joining
        attn_case("attn_decode_long", 8, 1, 1, 8000, 50000, 32, 8, 128, "f16", "token", 0.9, False, True),
        # drafts of a few tokens checked at once over prompts of any length, some empty
        attn_case("attn_draft_odd", 24, 1, 17, 0, 511, 12, 4, 80, "f16", "token", 0.8, True),
        # teacher-forced targets against long sources
        attn_case("attn_targets", 16, 512, 1024, 1024, 2048, 16, 4, 64, "bf16", "token"),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["int8", "norm", "attn"])
    if op == "int8":
        while True:
            M, K, N = log_int(rng, 1, 8192), log_int(rng, 32, 8192), log_int(rng, 16, 16384)
            if M * K * N <= 8192 * 4096 * 4096 and M * N <= 8192 * 8192:
                break
        c = int8_case("", M, K, N, rng.choice(["f32", "f16", "bf16"]), rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.5)
    elif op == "norm":
        while True:
            M, d = log_int(rng, 1, 65536), log_int(rng, 33, 16384)
            if M * d <= 65536 * 2048:
                break
        y = rng.choice(["f16", "bf16", "f32"])
        x = rng.choice(["f32", y])
        N = log_int(rng, 32, 4096) if y != "f32" and rng.random() < 0.4 and M * d <= 1 << 24 else 0
        c = norm_case("", M, d, x, y, rng.choice(["none", "scalar", "channel", "token"]), rng.random() < 0.5, rng.random() < 0.6,
                      rng.choice([1.0, 0.5, 0.70710678]), N)
    else:
        while True:
            B, q_hi, k_hi = log_int(rng, 1, 256), log_int(rng, 1, 1024), log_int(rng, 1, 50000)
            KVH, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 80, 96, 128])
            if B * q_hi * k_hi * KVH * G * D <= 16 * 1024 * 2048 * 16 * 64 and B * k_hi * KVH * D <= 8 * 50000 * 8 * 128:
                break
        c = attn_case("", B, rng.randint(0, q_hi) if B > 1 else q_hi, q_hi, rng.randint(0, k_hi) if B > 1 else k_hi, k_hi,
                      KVH * G, KVH, D, rng.choice(["f16", "bf16"]), rng.choice(["token", "head"]),
                      rng.choice([1.0, 1.0, 0.9, 0.5]), rng.random() < 0.3, rng.random() < 0.3, rng.randrange(1 << 20))
    del c["name"]
    return c


def lengths(case):
    """(query lengths, key lengths, first key row of each request, key rows)."""
    r = random.Random(case["lens"])
    B = case["B"]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(B)]
    k = [r.randint(case["k_lo"], case["k_hi"]) for _ in range(B)]
    q[0] = case["q_hi"]
    k[-1] = case["k_hi"]
    start, at = [], 0
    for n in k:
        start.append(at)
        at += case["k_hi"] if case["padded"] else n
    return q, k, start, at


def normal(shape, g, t=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case, "made_for": own}
    if case["op"] == "int8" or case.get("N"):
        K, N = case["K"] if case["op"] == "int8" else case["d"], case["N"]
        # weights as the library stores them: [N][K rounded up to 16] and a scale for each row
        s["w"] = torch.zeros((N, round_up(K, 16)), dtype=torch.int8, device="cuda")
        s["w"][:, :K] = (torch.randn((N, K), generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8)
        s["ws"] = (torch.rand(N, generator=g, device="cuda") * 1.5 + 0.5) * (1.0 / (40 * math.sqrt(K)))
        s["bias"] = normal((N,), g) if case.get("bias") else None
    if case["op"] == "int8":
        M, K = case["M"], case["K"]
        # activations whose channels have widths of their own, as behind a norm
        wide = torch.exp(normal((K,), g, scale=0.5))
        s["x"] = (normal((M, K), g) * wide).to(TYPES[case["x"]])
    elif case["op"] == "norm":
        M, d, ty = case["M"], case["d"], TYPES[case["y"]]
        s["x"] = normal((M, d), g, scale=2.0).to(TYPES[case["x"]])
        s["y"] = normal((M, d), g, scale=0.7).to(ty)
        s["post"] = normal((d,), g, scale=0.1) if case["post"] else None
        s["pre"] = normal((d,), g, scale=0.1)
        s["gate"] = {"none": lambda: None, "scalar": lambda: normal((1,), g), "channel": lambda: normal((d,), g),
                     "token": lambda: normal((M, d), g, ty)}[case["gate"]]()
    else:
        q, k, start, rows = lengths(case)
        H, KVH, D, t = case["H"], case["KVH"], case["D"], TYPES[case["type"]]
        s["q"] = normal((sum(q), H, D), g, t)
        if case["layout"] == "token":  # the two halves of a fused key and value projection
            kv = normal((max(rows, 1), 2, KVH, D), g, t)
            s["k"], s["v"] = kv[:, 0], kv[:, 1]
        else:  # one plane for each head
            kv = normal((2, KVH, max(rows, 1), D), g, t)
            s["k"], s["v"] = kv[0].transpose(0, 1), kv[1].transpose(0, 1)
        s["mask"] = None
        if case["keep"] < 1.0:
            s["mask"] = (torch.rand(max(rows, 1), generator=g, device="cuda") < case["keep"]).to(torch.uint8)
        s["scale"] = 1.0 / math.sqrt(D)
        if not own:
            lq, lk = torch.tensor(q, device="cuda"), torch.tensor(k, device="cuda")
            first = torch.cumsum(lq, 0) - lq
            jq, jk = torch.arange(max(q), device="cuda"), torch.arange(max(max(k), 1), device="cuda")
            s["q_in"], s["k_in"] = jq < lq[:, None], jk < lk[:, None]
            s["q_at"] = torch.where(s["q_in"], first[:, None] + jq, 0)
            s["k_at"] = torch.where(s["k_in"], torch.tensor(start, device="cuda")[:, None] + jk, 0)
    if own:
        n = needle()
        if "w" in s:
            M = case["M"]
            K = case["K"] if case["op"] == "int8" else case["d"]
            s["plan"] = n.Int8Plan(s["w"].data_ptr(), s["ws"].data_ptr(), K, case["N"], M)
            s["out"] = torch.empty((M, case["N"]), dtype=TYPES[case["y"]], device="cuda")
        if case["op"] == "norm":
            s["r"] = torch.empty_like(s["x"])
            if case["N"]:
                s["h"] = torch.empty((M, round_up(d, 16)), dtype=torch.int8, device="cuda")
                s["hs"] = torch.empty(M, device="cuda")
            else:
                s["h"] = torch.empty_like(s["y"])
        if case["op"] == "attn":
            q_start = [0] * len(q)
            for i in range(1, len(q)):
                q_start[i] = q_start[i - 1] + q[i - 1]
            s["plan"] = n.CrossAttnPlan(q_start, q, start, k, H, KVH, D, code(case["type"]))
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty((sum(q), H), device="cuda") if case["lse"] else None
    return s


def ptr(t):
    return None if t is None else t.data_ptr()


def quantized(x):
    """Rows of f32 as 8-bit values and their scales: scale = max|x| / 127, value = round(x * (127 / max|x|))."""
    top = x.abs().amax(dim=-1, keepdim=True)
    full = torch.full_like(top, 127.0)
    some = top >= 127.0 * 2.0 ** -126
    inv = torch.where(some, full / top, torch.zeros_like(top))
    return (x * inv).round().clamp(-127, 127), torch.where(some, top / full, torch.zeros_like(top))


def product(q, scale, s, K, out):
    y = (q @ s["w"][:, :K].float().t()) * (scale * s["ws"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(out)


def plain_norm(s, case):
    x, y = s["x"].float(), s["y"].float()
    if s["post"] is not None:
        y = y * (1.0 + s["post"]) / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = y * (torch.sigmoid(gate) if case["sigmoid"] else gate)
    r = case["scale"] * x + y
    h = r * (1.0 + s["pre"]) / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS)
    if case["N"]:
        return [r.to(TYPES[case["x"]]), product(*quantized(h), s, case["d"], TYPES[case["y"]])]
    return [r.to(TYPES[case["x"]]), h.to(TYPES[case["y"]])]


def plain_attn(s, case):
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G, B = H // KVH, case["B"]
    seen = s["k_in"]
    if s["mask"] is not None:
        seen = seen & (s["mask"][s["k_at"]] != 0)
    k, v = (torch.where(seen[..., None, None], t[s["k_at"]].float(), 0.0).transpose(1, 2) for t in (s["k"], s["v"]))
    q = s["q"][s["q_at"]].float().view(B, -1, KVH, G, D).permute(0, 2, 1, 3, 4).reshape(B, KVH, -1, D)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    x.masked_fill_(~seen[:, None, None, :], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(B, KVH, -1, G, D).permute(0, 2, 1, 3, 4).reshape(B, -1, H, D)[s["q_in"]].to(s["q"].dtype)
    if not case["lse"]:
        return [o]
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, float("-inf")))
    return [o, lse.view(B, KVH, -1, G).permute(0, 2, 1, 3).reshape(B, -1, H)[s["q_in"]]]


def run(s):
    case = s["case"]
    if own:
        n = needle()
        if case["op"] == "int8":
            s["plan"].matmul(s["x"].data_ptr(), case["M"], s["out"].data_ptr(), code(case["x"]), code(case["y"]), bias_ptr=ptr(s["bias"]))
            return [s["out"]]
        if case["op"] == "norm":
            flags = {"none": 0, "scalar": n.GATE_SCALAR, "channel": n.GATE_CHANNEL, "token": n.GATE_TOKEN}[case["gate"]]
            n.residual_norm(s["x"].data_ptr(), code(case["x"]), s["y"].data_ptr(), code(case["y"]), case["M"], case["d"],
                            s["pre"].data_ptr(), s["r"].data_ptr(), s["h"].data_ptr(), n.I8 if case["N"] else code(case["y"]),
                            post_scale_ptr=ptr(s["post"]), gate_ptr=ptr(s["gate"]),
                            gate_flags=flags | (n.GATE_SIGMOID if flags and case["sigmoid"] else 0),
                            residual_scale=case["scale"], h_scales_ptr=ptr(s.get("hs")))
            if not case["N"]:
                return [s["r"], s["h"]]
            s["plan"].matmul_quantized(s["h"].data_ptr(), s["hs"].data_ptr(), case["M"], s["out"].data_ptr(), code(case["y"]))
            return [s["r"], s["out"]]
        k, v = s["k"], s["v"]
        s["plan"].run(s["q"].data_ptr(), k.data_ptr(), v.data_ptr(), s["out"].data_ptr(), s["scale"],
                      k_strides=(k.stride(0), k.stride(1)), v_strides=(v.stride(0), v.stride(1)), key_mask_ptr=ptr(s["mask"]),
                      lse_ptr=ptr(s["lse"]))
        return [s["out"]] if s["lse"] is None else [s["out"], s["lse"]]
    if case["op"] == "int8":
        q, scale = quantized(s["x"].float())
        return [product(q, scale, s, case["K"], TYPES[case["y"]])]
    if case["op"] == "norm":
        return plain_norm(s, case)
    return plain_attn(s, case)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * size[case["x"]] + N * K + 4 * N * (2 if case["bias"] else 1) + M * N * size[case["y"]],
                "flops": 2.0 * M * K * N}
    if case["op"] == "norm":
        M, d, N, sx, sy = case["M"], case["d"], case["N"], size[case["x"]], size[case["y"]]
        b = M * d * (2 * sx + sy) + 4 * d * (2 if case["post"] else 1)
        b += {"none": 0, "scalar": 4, "channel": 4 * d, "token": M * d * sy}[case["gate"]]
        b += N * d + 4 * N + M * N * sy if N else M * d * sy
        return {"bytes": b, "flops": 2.0 * M * d * N + 12.0 * M * d}
    q, k, _, _ = lengths(case)
    H, KVH, D = case["H"], case["KVH"], case["D"]
    b = 2 * sum(q) * H * D * 2 + sum(n for n, m in zip(k, q) if m) * (2 * KVH * D * 2 + (case["keep"] < 1.0))
    return {"bytes": b + (sum(q) * H * 4 if case["lse"] else 0), "flops": 4.0 * H * D * sum(a * c for a, c in zip(q, k))}


def exact_product(h, s, w, K):
    """The 8-bit product in 64 bits; the rounding to 8 bits is of the f32 product x * (127 / max|x|)."""
    h = h.to(torch.float32)
    top = h.abs().max(dim=1).values
    inv = (127.0 / top.double()).float()
    ok = top.double() >= 127.0 * 2.0 ** -126
    q = torch.round((h.double() * inv.double()[:, None]).float()).double()
    q[~ok] = 0.0
    scale = torch.where(ok, top.double() / 127.0, 0.0)
    y = torch.einsum("mk,nk->mn", q, w[:, :K].double()) * scale[:, None] * s["ws"].double()[None]
    return y if s["bias"] is None else y + s["bias"].double()[None]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "int8":
        return [exact_product(s["x"], s, s["w"], case["K"])]
    if case["op"] == "norm":
        x, y = s["x"].double(), s["y"].double()
        if s["post"] is not None:
            y = y / y.pow(2).mean(1).add(EPS).sqrt()[:, None] * (s["post"].double() + 1)
        if s["gate"] is not None:
            gate = s["gate"].double()
            y = y * (1 / (1 + torch.exp(-gate)) if case["sigmoid"] else gate)
        r = x * case["scale"] + y
        h = r / r.pow(2).mean(1).add(EPS).sqrt()[:, None] * (s["pre"].double() + 1)
        return [r, exact_product(h, s, s["w"], case["d"]) if case["N"] else h]
    lq, lk, start, _ = lengths(case)
    H, KVH, D = case["H"], case["KVH"], case["D"]
    out = torch.zeros((sum(lq), H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(lq), H), float("-inf"), dtype=torch.float64, device="cuda")
    at = 0
    for n, m, first in zip(lq, lk, start):
        rows = slice(first, first + m)
        seen = torch.arange(first, first + m, device="cuda")
        if s["mask"] is not None:
            seen = seen[s["mask"][rows] != 0]
        if n and seen.numel():
            k, v = (t[seen].double().repeat_interleave(H // KVH, dim=1) for t in (s["k"], s["v"]))
            z = torch.einsum("qhd,khd->hqk", s["q"][at:at + n].double(), k) * s["scale"]
            lse[at:at + n] = torch.logsumexp(z, -1).t()
            out[at:at + n] = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v)
        at += n
    return [out, lse] if case["lse"] else [out]
