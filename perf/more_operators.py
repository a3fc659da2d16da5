"""Workloads of the 4-bit cache of keys and values and of the verification of drafts.

Each case is one step that a serving program makes around a decoder's cache:
new tokens are written in 4 bits and read back, a prefix is read back, query
rows attend to the cache, and drafted tokens are checked against the target's
logits.  `run` computes them in elementary torch operations, or, with `own`
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
GROUP = 32  # values of a head that share a scale and a minimum


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


def kv_case(name, op, B, new, length, H, KVH, D, t, page, causal=True, lse=False, lens=1):
    """B requests with new[0] to new[1] rows of this step and caches of length[0] to length[1] tokens (these rows
    among them where causal)."""
    return {"name": name, "op": op, "B": B, "new_lo": new[0], "new_hi": new[1], "len_lo": length[0], "len_hi": length[1],
            "H": H, "KVH": KVH, "D": D, "type": t, "page": page, "causal": causal, "lse": lse, "lens": lens}


def verify_case(name, B, lo, hi, V, t, probs, keep=1.0, greedy=0.0, lens=1):
    return {"name": name, "op": "verify", "B": B, "n_lo": lo, "n_hi": hi, "V": V, "type": t, "probs": probs, "keep": keep,
            "greedy": greedy, "lens": lens}


def listed():
    return [
        # a decode step of 64 requests of the shipped head shape: one token each, written and read back
        kv_case("store_step", "store", 64, (1, 1), (65, 512), 8, 4, 64, "bf16", 64),
        # prompts of any length at once, pages of 16, a head size that does not fill its last group
        kv_case("store_odd", "store", 33, (1, 777), (1, 1500), 12, 4, 80, "f16", 16),
        # a prefill batch
        kv_case("store_prefill", "store", 16, (2048, 2048), (2048, 8192), 32, 8, 128, "bf16", 64),
        # one request's prompt, read back for a kernel that takes 16 bits
        kv_case("read_prompt", "read", 1, (500, 500), (500, 500), 8, 4, 64, "bf16", 64),
        # long documents, read back whole
        kv_case("read_long", "read", 8, (8000, 50000), (8000, 50000), 32, 8, 128, "f16", 128),
        # one decode step of 256 requests over their prompts' encoder states
        kv_case("attn_decode_256", "attn", 256, (1, 1), (64, 512), 8, 4, 64, "bf16", 64, False),
        # a decode step over few long documents, the row statistics kept for joining
        kv_case("attn_decode_long", "attn", 8, (1, 1), (8000, 50000), 32, 8, 128, "f16", 128, True, True),
        # drafts of a few tokens checked at once over caches of any length, pages of 16
        kv_case("attn_draft_odd", "attn", 24, (1, 9), (9, 2000), 12, 4, 80, "f16", 16),
        # a chunk of each of four long prompts
        kv_case("attn_chunk", "attn", 4, (1024, 1024), (4096, 16384), 32, 8, 128, "bf16", 64),
        # one request's four drafts under a constraint, the shipped vocabulary
        verify_case("verify_one", 1, 4, 4, 8192, "f32", True, 0.05),
        # requests with up to five drafts, some greedy, by a drafter that gives no probabilities
        verify_case("verify_odd", 96, 0, 5, 32003, "f16", False, 0.5, 0.3),
        # a large batch over a large vocabulary
        verify_case("verify_batch", 256, 4, 4, 131072, "bf16", True),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attn", "attn", "verify"])
    if op == "verify":
        while True:
            B, hi, V = log_int(rng, 1, 256), rng.randint(0, 8), log_int(rng, 100, 160000)
            if B * (hi + 1) * V <= 256 * 5 * 131072:
                break
        c = verify_case("", B, rng.randint(0, hi), hi, V, rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.6,
                        rng.choice([1.0, 0.5, 0.05]), rng.choice([0.0, 0.0, 0.3, 1.0]), rng.randrange(1 << 20))
        del c["name"]
        return c
    page, t = rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"])
    while True:
        B, n_hi, k_hi = log_int(rng, 1, 256), log_int(rng, 1, 1024), log_int(rng, 1, 50000)
        KVH, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 40, 64, 80, 96, 128])
        k_hi = max(n_hi, k_hi)
        if op == "attn":
            if B * n_hi * k_hi * KVH * G * D > 4 * 1024 * 16384 * 32 * 128 or B * n_hi * k_hi * KVH * G > 1 << 31:
                continue
        if op == "store" and B * n_hi * KVH * D > 16 * 2048 * 8 * 128:
            continue
        if B * k_hi * KVH * D <= 8 * 50000 * 8 * 128:
            break
    new, length = (rng.randint(0, n_hi) if B > 1 else n_hi, n_hi), (rng.randint(0, k_hi) if B > 1 else k_hi, k_hi)
    if op == "read":
        new = length
    c = kv_case("", op, B, new, length, KVH * G, KVH, D, t, page, op != "attn" or rng.random() < 0.6,
                op == "attn" and rng.random() < 0.4, rng.randrange(1 << 20))
    del c["name"]
    return c


def lengths(case):
    """(rows of this step, cached tokens) of each request."""
    r = random.Random(case["lens"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    total = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["B"])]
    new[0], total[-1] = case["new_hi"], case["len_hi"]
    if case["op"] == "read":
        new = total
    elif case["causal"]:
        total = [max(a, b) for a, b in zip(new, total)]
    return new, total


def drafts(case):
    r = random.Random(case["lens"])
    n = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]
    n[0] = case["n_hi"]
    return n, [0.0 if r.random() < case["greedy"] else r.choice([0.7, 1.0, 1.3]) for _ in n]


def starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def keys_and_values(rows, case, g):
    """Keys whose channels have widths and offsets of their own, as caches have them; values."""
    KVH, D, t = case["KVH"], case["D"], TYPES[case["type"]]
    wide, at = torch.exp(0.5 * normal((KVH, D), g)), normal((KVH, D), g)
    # parts of the rows that a fused projection writes
    kv = torch.empty((max(rows, 1), 2, KVH, D), dtype=t, device="cuda")
    kv[:, 0] = normal((max(rows, 1), KVH, D), g).mul_(wide).add_(at)
    kv[:, 1] = normal((max(rows, 1), KVH, D), g)
    return kv[:rows, 0], kv[:rows, 1]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return prepare_verify(case, g) if case["op"] == "verify" else prepare_kv(case, g, seed)


def prepare_kv(case, g, seed):
    B, H, KVH, D, page, t = (case[k] for k in ("B", "H", "KVH", "D", "page", "type"))
    new, total = lengths(case)
    s = {"case": case, "new": new, "total": total}
    if case["op"] == "store":
        s["k"], s["v"] = keys_and_values(sum(new), case, g)
    else:
        k, v = keys_and_values(sum(total), case, g)
    if case["op"] == "attn":
        s["q"] = normal((sum(new), H, D), g).to(TYPES[t])
        s["scale"] = 1.0 / math.sqrt(D)
    if own:
        n = needle()
        used = [(m + page - 1) // page for m in total]
        order = list(range(sum(used)))
        random.Random(seed).shuffle(order)  # a pool's pages come in any order
        width = max(max(used), 1)
        at = starts(used)
        table = i32([order[at[i]:at[i + 1]] + [-1] * (width - used[i]) for i in range(B)])
        n_pages = max(sum(used), 1)
        s["plan"] = n.Kv4Plan(H, KVH, D, page, n_pages, B, max(sum(new), sum(total), 1), code(t))
        s["pages"] = torch.empty(n_pages * n.kv4_page_bytes(KVH, D, page), dtype=torch.uint8, device="cuda")
        s["held"] = [table, i32(starts(new)), i32(total), i32(starts(total))]
        s["batch"] = n.Kv4Batch(s["held"][1].data_ptr(), s["held"][2].data_ptr(), table.data_ptr(), B, sum(new), width, max(new))
        if case["op"] == "attn":
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty((sum(new), H), device="cuda") if case["lse"] else None
        else:
            s["out"] = [torch.empty((sum(new), KVH, D), dtype=TYPES[t], device="cuda") for _ in range(2)]
        if case["op"] != "store":
            whole = n.Kv4Batch(s["held"][3].data_ptr(), s["held"][2].data_ptr(), table.data_ptr(), B, sum(total), width, max(total))
            s["plan"].append(s["pages"].data_ptr(), whole, k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2])
            torch.cuda.synchronize()
    elif case["op"] != "store":
        s["cache"] = quantised(k), quantised(v)
    if not own and case["op"] == "attn":
        lk, lq = i32(total).long(), i32(new).long()
        first, at = torch.cumsum(lq, 0) - lq, torch.cumsum(lk, 0) - lk
        jq, jk = torch.arange(max(max(new), 1), device="cuda"), torch.arange(max(max(total), 1), device="cuda")
        s["q_in"], k_in = jq < lq[:, None], jk < lk[:, None]
        s["q_at"], s["k_at"] = torch.where(s["q_in"], first[:, None] + jq, 0), torch.where(k_in, at[:, None] + jk, 0)
        s["limit"] = (lk - lq)[:, None] + jq if case["causal"] else (lk - 1)[:, None].expand(B, len(jq))
    return s


def prepare_verify(case, g):
    B, V, t = case["B"], case["V"], TYPES[case["type"]]
    n, temps = drafts(case)
    rows, total = sum(n) + B, sum(n)
    s = {"case": case, "n": n, "temps": temps}
    # a few likely tokens in each row, the rest behind them
    z = normal((rows, V), g).mul_(2.0)
    z.scatter_add_(1, torch.randint(0, V, (rows, 4), generator=g, device="cuda"), 6.0 + 2.0 * normal((rows, 4), g))
    s["logits"] = z.to(t)
    allowed = None
    s["mask"] = None
    if case["keep"] < 1.0:  # bit v % 64 of word v / 64, as the constrained decoder gives them
        words = (V + 63) // 64
        allowed = torch.zeros((rows, words * 64), dtype=torch.bool, device="cuda")
        allowed[:, :V] = torch.rand((rows, V), generator=g, device="cuda") < case["keep"]
        allowed.scatter_(1, torch.randint(0, V, (rows, 1), generator=g, device="cuda"), True)
        weight = torch.ones(64, dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
        s["mask"] = (allowed.view(rows, words, 64) * weight).sum(-1)
    # the drafter's distribution is near the target's; its drafts come from it
    first = starts([m + 1 for m in n])
    of = torch.tensor([first[i] + j for i in range(B) for j in range(n[i])], dtype=torch.long, device="cuda")
    s["ids"] = torch.zeros(max(total, 1), dtype=torch.int32, device="cuda")
    s["probs"] = torch.zeros((max(total, 1), V), device="cuda") if case["probs"] else None
    for a in range(0, total, 256):
        rows_ = of[a:a + 256]
        d = s["logits"][rows_].float() + 0.7 * normal((len(rows_), V), g)
        if allowed is not None:
            d.masked_fill_(~allowed[rows_, :V], float("-inf"))
        if case["probs"]:
            d = torch.softmax(d, -1)
            s["probs"][a:a + 256] = d
            s["ids"][a:a + 256] = torch.multinomial(d, 1, generator=g)[:, 0].int()
        else:
            s["ids"][a:a + 256] = d.argmax(-1).int()
    s["u"] = torch.rand(max(total, 1), generator=g, device="cuda")
    s["final"] = torch.rand(B, generator=g, device="cuda")
    s["T"] = torch.tensor(temps, device="cuda")
    s["width"] = max(n) + 1
    if own:
        nb = needle()
        s["start"] = i32(starts(n))
        s["plan"] = nb.VerifyPlan(V, B, max(total, 1), code(case["type"]))
        s["out"] = torch.empty((B, s["width"]), dtype=torch.int32, device="cuda")
        s["len"] = torch.empty(B, dtype=torch.int32, device="cuda")
        s["logp"] = torch.empty((B, s["width"]), device="cuda")
    else:
        s["row"] = torch.tensor([i for i in range(B) for _ in range(n[i] + 1)], device="cuda")
        j = torch.arange(s["width"], device="cuda")
        nn = torch.tensor(n, device="cuda")
        s["has"] = j < nn[:, None]
        s["first"] = torch.tensor(first[:-1], device="cuda")
        s["draft_at"] = torch.where(s["has"], torch.tensor(starts(n)[:-1], device="cuda")[:, None] + j, 0)
        s["nn"] = nn
    return s


def ptr(t):
    return None if t is None else t.data_ptr()


def run(s):
    case = s["case"]
    if case["op"] == "verify":
        if not own:
            return plain_verify(s)
        s["plan"].run(s["logits"].data_ptr(), s["start"].data_ptr(), s["ids"].data_ptr(), s["u"].data_ptr(), s["final"].data_ptr(),
                      s["out"].data_ptr(), s["len"].data_ptr(), case["B"], sum(s["n"]), s["width"], draft_probs_ptr=ptr(s["probs"]),
                      temperature_ptr=s["T"].data_ptr(), mask_ptr=ptr(s["mask"]), logprobs_ptr=s["logp"].data_ptr())
        return [s["out"], s["len"], s["logp"]]
    if not own:
        return {"store": plain_store, "read": plain_read, "attn": plain_attn}[case["op"]](s)
    pages = s["pages"].data_ptr()
    if case["op"] == "attn":
        s["plan"].attn(pages, s["batch"], s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], causal=case["causal"], lse_ptr=ptr(s["lse"]))
        return [s["out"]] if s["lse"] is None else [s["out"], s["lse"]]
    if case["op"] == "store":
        k, v = s["k"], s["v"]
        s["plan"].append(pages, s["batch"], k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2])
    s["plan"].read(pages, s["batch"], s["out"][0].data_ptr(), s["out"][1].data_ptr())
    return s["out"]


def quantised(x):
    """Values of a row's head in groups of 32, 4 bits each: (codes, scales, minima).

    minimum = f16(min x), scale = f16((max x - min x) / 15), code = rint((x - minimum) * (1 / scale)) within 0 to 15;
    scales and minima are one half each, all else is rounded to f32."""
    codes, scales, minima = [], [], []
    for a in range(0, x.shape[-1], GROUP):
        v = x[..., a:a + GROUP].float()
        lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        scale, least = ((hi - lo) / 15.0).half(), lo.half()
        inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(lo))
        codes.append(((v - least.float()) * inv).round().clamp(0, 15).to(torch.uint8))
        scales.append(scale[..., 0])
        minima.append(least[..., 0])
    return torch.cat(codes, -1), torch.stack(scales, -1), torch.stack(minima, -1)


def values(codes, scales, minima, rows=None):
    if rows is not None:
        codes, scales, minima = codes[rows], scales[rows], minima[rows]
    D = codes.shape[-1]
    scales, minima = (t.float().repeat_interleave(GROUP, -1)[..., :D] for t in (scales, minima))
    return codes.float() * scales + minima


def plain_store(s):
    return [values(*quantised(s[n])).to(s[n].dtype) for n in ("k", "v")]


def plain_read(s):
    t = TYPES[s["case"]["type"]]
    return [values(*c).to(t) for c in s["cache"]]


def plain_attn(s):
    case = s["case"]
    H, KVH, D, B = case["H"], case["KVH"], case["D"], case["B"]
    G, out, lse = H // KVH, [], []
    # a few requests at a time: their rows and keys padded to the longest
    step = max(1, (1 << 31) // (max(max(s["new"]), 1) * max(max(s["total"]), 1) * H + 2 * max(max(s["total"]), 1) * KVH * D))
    for a in range(0, B, step):
        b = slice(a, a + step)
        nq, nk = max(max(s["new"][b]), 1), max(max(s["total"][b]), 1)
        k, v = (values(*c, s["k_at"][b, :nk]).transpose(1, 2) for c in s["cache"])
        seen = torch.arange(nk, device="cuda") <= s["limit"][b, :nq, None]
        q_in = s["q_in"][b, :nq]
        n = len(q_in)
        q = s["q"][s["q_at"][b, :nq]].float().view(n, nq, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(n, KVH, G * nq, D)
        x = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).view(n, KVH, G, nq, nk)
        x.masked_fill_(~seen[:, None, None], float("-inf"))
        top = x.amax(-1, keepdim=True)
        x.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
        total = x.sum(-1, keepdim=True)
        # keys behind a request's are not there
        v = torch.where((torch.arange(nk, device="cuda") < i32(s["total"][b])[:, None])[:, None, :, None], v, 0.0)
        o = torch.matmul(x.view(n, KVH, G * nq, nk), v).view(n, KVH, G, nq, D)
        o = o / torch.where(total > 0, total, torch.ones_like(total))
        out.append(o.permute(0, 3, 1, 2, 4).reshape(n, nq, H, D)[q_in].to(s["q"].dtype))
        if case["lse"]:
            l = torch.where(total > 0, top + torch.log(total), torch.full_like(total, float("-inf")))
            lse.append(l[..., 0].permute(0, 3, 1, 2).reshape(n, nq, H)[q_in])
    return [torch.cat(out)] + ([torch.cat(lse)] if case["lse"] else [])


def bits(mask, V):
    """The allowed entries that bitmaps of 64-bit words stand for."""
    b = (mask[..., None] >> torch.arange(64, device=mask.device)) & 1
    return b.flatten(-2)[..., :V] != 0


def plain_verify(s):
    """In 64 bits: a token is where a cumulative sum passes a random number."""
    case = s["case"]
    B, V, n = case["B"], case["V"], s["nn"]
    logits, T = s["logits"], s["T"].double()
    greedy = T <= 0
    cut = torch.where(greedy, torch.ones_like(T), T)
    rows = logits.shape[0]
    best, top, total = (torch.empty(rows, dtype=d, device="cuda") for d in (torch.int64, torch.float64, torch.float64))
    picked = torch.zeros(rows, dtype=torch.float64, device="cuda")
    has, at = s["has"], s["first"][:, None] + torch.arange(s["width"], device="cuda")
    draft = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    draft[at[has]] = s["ids"][s["draft_at"][has]].long()

    def scores(r):
        z = logits[r].double() / cut[s["row"][r], None]
        return z if s["mask"] is None else torch.where(bits(s["mask"][r], V), z, float("-inf"))

    for a in range(0, rows, 128):
        r = torch.arange(a, min(a + 128, rows), device="cuda")
        z = scores(r)
        top[r] = z.amax(-1)
        best[r] = torch.where(z == top[r, None], torch.arange(V, device="cuda"), V).amin(-1)
        w = torch.exp(z - top[r, None])
        total[r] = w.sum(-1)
        picked[r] = w.gather(1, draft[r, None].clamp(min=0))[:, 0]
    p = torch.where(has, (picked / total)[torch.where(has, at, 0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    ids = s["ids"].long()[s["draft_at"]]
    q = torch.ones_like(p) if s["probs"] is None else s["probs"][s["draft_at"], ids].double()
    won = torch.where(greedy[:, None], best[torch.where(has, at, 0)] == ids, s["u"][s["draft_at"]].double() * q < p) & has
    taken = torch.cumprod(won.long(), 1).sum(1)
    row, reject = s["first"] + taken, taken < n
    final, final_logp = best[row].clone(), torch.empty(B, dtype=torch.float64, device="cuda")
    for a in range(0, B, 128):
        i = torch.arange(a, min(a + 128, B), device="cuda")
        r = row[i]
        z = scores(r) - top[r, None]
        p = torch.exp(z) / total[r, None]
        d = s["draft_at"][i, torch.clamp(taken[i], max=s["width"] - 1)]
        if s["probs"] is None:
            rest = p.scatter(1, s["ids"].long()[d, None], 0.0)
        else:
            rest = torch.clamp(p - s["probs"][d].double(), min=0.0)
        rest = torch.where((reject[i] & (rest.sum(-1) > 0))[:, None], rest, p)
        c = torch.cumsum(rest, -1)
        past = c > s["final"][i, None].double() * c[:, -1:]
        last = torch.where(rest > 0, torch.arange(V, device="cuda"), -1).amax(-1)
        pick = torch.where(past & (rest > 0), torch.arange(V, device="cuda"), V).amin(-1)
        final[i] = torch.where(greedy[i], final[i], torch.where(pick < V, pick, last))
        final_logp[i] = z.gather(1, final[i, None])[:, 0] - torch.log(total[r])
    j = torch.arange(s["width"], device="cuda")
    out = torch.where(j < taken[:, None], ids, torch.where(j == taken[:, None], final[:, None], -1))
    # the log-probability of each token in its row
    logp = torch.log(picked / total)[torch.where(has, at, 0)]
    logp = torch.where(j < taken[:, None], logp, torch.where(j == taken[:, None], final_logp[:, None], 0.0))
    return [out.int(), (taken + 1).int(), logp.float()]


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["op"] == "verify":
        n, _ = drafts(case)
        rows, V, B = sum(n) + case["B"], case["V"], case["B"]
        mask = (V + 63) // 64 * 8 if case["keep"] < 1.0 else 0
        # the drafter's probabilities: of each draft's token (a rejected row's others are read as the data have it)
        return {"bytes": rows * (V * size + mask) + sum(n) * (8 + 4 * case["probs"]) + B * (8 + 4 + 8 * (max(n) + 1)), "flops": 4.0 * rows * V}
    new, total = lengths(case)
    H, KVH, D = case["H"], case["KVH"], case["D"]
    token = 2 * KVH * (D // 2 + (D + GROUP - 1) // GROUP * 4)  # a token's codes, scales and minima
    wide = 2 * KVH * D * size
    if case["op"] == "store":
        return {"bytes": sum(new) * (wide + token + token + wide), "flops": 8.0 * sum(new) * 2 * KVH * D}
    if case["op"] == "read":
        return {"bytes": sum(total) * (token + wide), "flops": 2.0 * sum(total) * 2 * KVH * D}
    pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(new, total))
    b = 2 * sum(new) * H * D * size + sum(b for a, b in zip(new, total) if a) * token + (sum(new) * H * 4 if case["lse"] else 0)
    return {"bytes": b, "flops": 4.0 * H * D * pairs}


def exact_values(x):
    """What 4 bits leave of x, in 64 bits; the code's rounding is of f32 quantities."""
    n = x.shape[-1]
    y = torch.zeros((*x.shape[:-1], (n + 31) // 32 * 32), dtype=torch.float64, device=x.device)
    y[..., :n] = x.double()
    y = y.unflatten(-1, (-1, 32))
    there = (torch.arange(y.shape[-2] * 32, device=x.device) < n).view(-1, 32)
    low, high = torch.where(there, y, math.inf).min(-1).values, torch.where(there, y, -math.inf).max(-1).values
    step = ((high - low).float().double() / 15).float().to(torch.float16)
    base = low.float().to(torch.float16).double()
    over = torch.where(step > 0, (1 / step.double()).float().double(), 0.0)
    t = ((y - base[..., None]).float().double() * over[..., None]).float()
    t = torch.round(t.double()).clamp(0, 15)
    return (base[..., None] + step.double()[..., None] * t).flatten(-2)[..., :n]


def exact(case, seed):
    global own
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "verify":
        kept, own = own, False
        try:
            s = prepare_verify(case, g)
        finally:
            own = kept
        return exact_verify(s)
    new, total = lengths(case)
    k, v = keys_and_values(sum(new if case["op"] == "store" else total), case, g)
    if case["op"] != "attn":
        return [exact_values(k), exact_values(v)]
    H, KVH, D = case["H"], case["KVH"], case["D"]
    q = normal((sum(new), H, D), g).to(TYPES[case["type"]])
    out = torch.zeros((sum(new), H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), H), float("-inf"), dtype=torch.float64, device="cuda")
    qa, ka = starts(new), starts(total)
    for i, (m, n) in enumerate(zip(new, total)):
        if not m or not n:
            continue
        kk, vv = (exact_values(t[ka[i]:ka[i + 1]]) for t in (k, v))
        for h in range(H):
            for a in range(0, m, 512):
                rows = torch.arange(a, min(a + 512, m), device="cuda")
                z = q[qa[i] + rows, h].double() @ kk[:, h * KVH // H].t() / math.sqrt(D)
                if case["causal"]:
                    z[torch.arange(n, device="cuda")[None] > (rows + n - m)[:, None]] = float("-inf")
                lse[qa[i] + rows, h] = torch.logsumexp(z, -1)
                out[qa[i] + rows, h] = torch.softmax(z, -1) @ vv[:, h * KVH // H]
    return [out, lse] if case["lse"] else [out]


def exact_verify(s):
    """One request after another, each row when it is reached."""
    case, V = s["case"], s["case"]["V"]
    out = torch.full((case["B"], s["width"]), -1, dtype=torch.int32, device="cuda")
    logp = torch.zeros((case["B"], s["width"]), dtype=torch.float64, device="cuda")
    lens, at, draft = [], 0, 0
    ids, u, final = s["ids"].tolist(), s["u"].tolist(), s["final"].tolist()
    shift = torch.arange(64, device="cuda")
    for i, (n, T) in enumerate(zip(s["n"], s["temps"])):
        for j in range(n + 1):
            z = s["logits"][at + j].double()
            if s["mask"] is not None:
                open_ = ((s["mask"][at + j][:, None] >> shift) % 2 != 0).flatten()[:V]
                z = z.masked_fill(~open_, float("-inf"))
            if T == 0:
                token = int((z == z.max()).nonzero()[0])
                ok = j < n and ids[draft + j] == token
            else:
                # the temperature is an f32 number
                p = torch.softmax(z / float(torch.tensor(T)), 0)
                rest = p
                ok = False
                if j < n:
                    d = ids[draft + j]
                    q = torch.zeros_like(p) if s["probs"] is None else s["probs"][draft + j].double()
                    if s["probs"] is None:
                        q[d] = 1.0
                    ok = u[draft + j] * float(q[d]) < float(p[d])
                    left = (p - q).clamp(min=0)
                    rest = left if float(left.sum()) > 0 else p
                if not ok:
                    c = rest.cumsum(0)
                    token = int(torch.searchsorted(c, c[-1] * final[i], right=True).clamp(max=int(rest.nonzero()[-1])))
            out[i, j] = ids[draft + j] if ok else token
            logp[i, j] = torch.log_softmax(z if T == 0 else z / float(torch.tensor(T)), 0)[out[i, j].long()]
            if not ok:
                break
        lens.append(j + 1)
        at, draft = at + n + 1, draft + n
    return [out, i32(lens), logp]
