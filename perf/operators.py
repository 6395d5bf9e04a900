"""Cases of the attention operators: head norms with the position rotation
(norm_rope), attention over packed prompts (attention_packed) and attention of
a batch whose requests share a long prefix (attention_prefix).

`run` computes a case with elementary torch operations in 32 bits, or, where
`own` is true, through mlk2_b200.api. `exact` computes it in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------

def listed():
    return [
        # norm_rope. One decode step of a small batch: latency.
        norm_rope_case("norm_rope decode 16 tokens bf16", tokens=16, heads=32, kv_heads=8, d=128),
        # A packed prompt batch of odd length, q and k as slices of one projection.
        norm_rope_case("norm_rope prompt 5003 tokens bf16", tokens=5003, heads=32, kv_heads=8, d=128),
        # Image patches: no norm weights, three position axes over d = 80, neighbouring pairs.
        norm_rope_case("norm_rope patches 9801 tokens f16", tokens=9801, heads=16, kv_heads=16, d=80,
                       axes=3, interleaved=True, norm=False, dtype="f16"),
        # A training-sized pass over many prompts, half of each head rotated.
        norm_rope_case("norm_rope 65536 tokens f16", tokens=65536, heads=16, kv_heads=2, d=128, rot=64,
                       dtype="f16"),
        # attention_packed. A single short question: latency.
        packed_case("packed one prompt of 17 f16", seqs=1, total=17, heads=8, kv_heads=2, d=64, dtype="f16"),
        # A prompt batch of very different lengths, with rows of padding behind the last.
        packed_case("packed 9 prompts in 6011 bf16", seqs=9, total=6011, heads=32, kv_heads=8, d=128,
                    pad=37),
        # Patches of three images: every patch sees its whole image.
        packed_case("packed 3 images in 4107 f16", seqs=3, total=4107, heads=16, kv_heads=16, d=80,
                    causal=False, dtype="f16"),
        # The next pieces of prompts whose earlier keys are there already.
        packed_case("packed pieces 1030 after 7000 bf16", seqs=5, total=1030, history=7000, heads=32,
                    kv_heads=4, d=128),
        # One long prompt.
        packed_case("packed one prompt of 8192 f16", seqs=1, total=8192, heads=32, kv_heads=8, d=128,
                    dtype="f16"),
        # attention_prefix. A few requests behind a short common instruction: latency.
        prefix_case("prefix 501 batch 4 f16", batch=4, steps=1, prefix=501, longest=61, heads=8, kv_heads=2,
                    d=64, page=0, dtype="f16"),
        # Drafted tokens of a batch, five a request, checked in one pass.
        prefix_case("prefix 2003 batch 24 by 5 bf16", batch=24, steps=5, prefix=2003, longest=700, heads=16,
                    kv_heads=4, d=128, page=16),
        # A serving batch behind one long document.
        prefix_case("prefix 32768 batch 80 bf16", batch=80, steps=1, prefix=32768, longest=2048, heads=32,
                    kv_heads=8, d=128, page=64),
    ]


def norm_rope_case(name, tokens, heads, kv_heads, d, rot=0, axes=1, interleaved=False, norm=True,
                   dtype="bf16"):
    return {"name": name, "op": "norm_rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "d": d, "rot": rot or d, "axes": axes, "interleaved": interleaved, "norm": norm,
            "dtype": dtype}


def packed_case(name, seqs, total, heads, kv_heads, d, history=0, pad=0, causal=True, dtype="bf16"):
    return {"name": name, "op": "packed", "seqs": seqs, "total": total, "history": history, "pad": pad,
            "heads": heads, "kv_heads": kv_heads, "d": d, "causal": causal, "dtype": dtype}


def prefix_case(name, batch, steps, prefix, longest, heads, kv_heads, d, page, dtype="bf16"):
    return {"name": name, "op": "prefix", "batch": batch, "steps": steps, "prefix": prefix,
            "longest": longest, "heads": heads, "kv_heads": kv_heads, "d": d, "page": page,
            "dtype": dtype}


def draw(rng):
    """A case of the same ranges: lengths over their logarithm, odd ones among them."""
    op = rng.choice(["norm_rope", "packed", "prefix"])
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    dtype = rng.choice(["f16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "norm_rope":
        d = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([d, d // 2 // 16 * 16])
        most = 65536 * 18 * 128 // ((group + 1) * kv_heads * d)
        c = norm_rope_case("", spread(1, min(65536, most)), group * kv_heads, kv_heads, d, rot,
                           rng.choice([1, 1, 2, 3]), rng.random() < 0.3, rng.random() < 0.7, dtype)
    elif op == "packed":
        d = rng.choice([64, 80, 96, 128])
        total = spread(1, 6000)
        causal = rng.random() < 0.7
        history = spread(1, 4000) if causal and rng.random() < 0.4 else 0
        c = packed_case("", rng.randint(1, min(16, total)), total, group * kv_heads, kv_heads, d, history,
                        rng.choice([0, 0, 11]), causal, dtype)
        while c["heads"] * total * (total + history) > 32 * 8192 * 4096:
            c["kv_heads"] = max(1, c["kv_heads"] // 2)
            c["heads"] = c["kv_heads"] * group
            total = c["total"] = max(c["seqs"], total * 3 // 4)
    else:
        c = prefix_case("", spread(1, 80), rng.choice([1, 1, 1, 2, 5]), spread(1, 20000), spread(8, 1500),
                        group * kv_heads, kv_heads, rng.choice([64, 80, 96, 128]),
                        rng.choice([0, 16, 64, 128]), dtype)
        c["longest"] = max(c["longest"], c["steps"])
        while c["batch"] * c["steps"] * c["heads"] * (c["prefix"] + c["longest"]) > 80 * 32 * 33000:
            c["batch"] = max(1, c["batch"] // 2)
            c["prefix"] = max(1, c["prefix"] * 3 // 4)
    del c["name"]
    return c


def packed_lengths(case):
    """(queries, keys) of each sequence, from the case alone: uneven shares of the total."""
    r = random.Random("%d of %d" % (case["seqs"], case["total"]))

    def shares(total, least):
        cuts = sorted(r.sample(range(1, total), case["seqs"] - 1)) if least and case["seqs"] > 1 else \
            sorted(r.randint(0, total) for _ in range(case["seqs"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [total])]

    q = shares(case["total"], 1)
    return q, [a + h for a, h in zip(q, shares(case["history"], 0))]


def prefix_lengths(case):
    """Keys of each request behind the prefix, its new tokens among them; the first has the longest."""
    r = random.Random("%d of %d" % (case["batch"], case["longest"]))
    return [case["longest"]] + [r.randint(case["steps"], case["longest"]) for _ in range(case["batch"] - 1)]


def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "norm_rope":
        t, elems = case["tokens"], case["tokens"] * (h + kv) * d
        table = 4 * case["rot"] * min(t, table_rows(case))  # each table row once
        return {"bytes": 2 * 2 * elems + 4 * t * case["axes"] + table + (4 * d if case["norm"] else 0),
                "flops": 7 * elems}
    if case["op"] == "packed":
        q, k = packed_lengths(case)
        if case["causal"]:  # query i of a sequence sees its keys up to i + keys - queries
            pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(q, k))
        else:
            pairs = sum(a * b for a, b in zip(q, k))
        return {"bytes": 2 * 2 * d * (h * sum(q) + kv * sum(k)) + 8 * (len(q) + 1),
                "flops": 4 * d * h * pairs}
    lens, t, b = prefix_lengths(case), case["steps"], case["batch"]
    seen = sum(t * (n - t) + t * (t + 1) // 2 for n in lens)
    return {"bytes": 2 * 2 * d * (h * b * t + kv * (case["prefix"] + sum(lens))) + 4 * b,
            "flops": 4 * d * h * (b * t * case["prefix"] + seen)}


# ---- inputs -------------------------------------------------------------------

def table_rows(case):
    return 32768 if case["axes"] == 1 else 512  # positions of a context, or of one image axis


def sections(case):
    """How many rotated pairs each position axis has."""
    half, n = case["rot"] // 2, case["axes"]
    return [half - (n - 1) * (half // n)] + [half // n] * (n - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    h, kv, d = case["heads"], case["kv_heads"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "norm_rope":
        t = case["tokens"]
        qkv = normal(t, h + 2 * kv, d)  # one projection's output: q, k and v heads side by side
        if case["axes"] == 1:
            pos = (torch.arange(t, device="cuda") + seed % 97) % table_rows(case)
        else:  # frames of 17 by 23 patches
            at = torch.arange(t, device="cuda")
            pos = torch.stack([at // (17 * 23), at // 23 % 17, at % 23][:case["axes"]])
        # The angles of far positions are formed in 64 bits; the table is rounded once.
        freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        angle = torch.arange(table_rows(case), device="cuda", dtype=torch.float64)[:, None] * freq
        table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        return {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "positions": pos.to(torch.int32),
                "table": table, "sections": sections(case),
                "axis": torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(sections(case))).cuda(),
                "q_weight": (1 + 0.2 * normal(d).float()).to(dt) if case["norm"] else None,
                "k_weight": (1 + 0.2 * normal(d).float()).to(dt) if case["norm"] else None,
                "q_out": torch.zeros((t, h, d), dtype=dt, device="cuda"),
                "k_out": torch.zeros((t, kv, d), dtype=dt, device="cuda")}
    if case["op"] == "packed":
        nq, nk = packed_lengths(case)
        starts = lambda n: ints([0] + torch.tensor(n).cumsum(0).tolist())  # noqa: E731
        rows = case["total"] + case["pad"]
        return {"case": case, "q": normal(rows, h, d), "k": normal(sum(nk), kv, d),
                "v": normal(sum(nk), kv, d), "q_starts": starts(nq), "k_starts": starts(nk),
                "y": torch.zeros((rows, h, d), dtype=dt, device="cuda")}
    b, page = case["batch"], case["page"] or case["longest"]
    lens = prefix_lengths(case)
    wide = -(-case["longest"] // page)
    s = {"case": case, "q": normal(b, case["steps"], h, d), "prefix_k": normal(case["prefix"], kv, d),
         "prefix_v": normal(case["prefix"], kv, d), "lens": ints(lens), "pages": None,
         "k_pages": normal(b * wide, page, kv, d), "v_pages": normal(b * wide, page, kv, d),
         "y": torch.zeros((b, case["steps"], h, d), dtype=dt, device="cuda")}
    if case["page"]:  # pages in the order in which a server happened to hand them out
        s["pages"] = torch.randperm(b * wide, generator=g, device="cuda").view(b, wide).to(torch.int32)
    return s


# ---- the operators --------------------------------------------------------------

def run(s):
    case = s["case"]
    scale = case["d"] ** -0.5
    if own:
        from mlk2_b200 import api

        if case["op"] == "norm_rope":
            api.norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], s["table"], s["positions"],
                          sections=s["sections"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                          eps=1e-6, interleaved=case["interleaved"])
            return s["q_out"], s["k_out"]
        if case["op"] == "packed":
            api.attention_packed(s["q"], s["k"], s["v"], s["y"], s["q_starts"], s["k_starts"], scale,
                                 causal=case["causal"])
            return s["y"]
        api.attention_prefix(s["q"], s["prefix_k"], s["prefix_v"], s["k_pages"], s["v_pages"], s["y"],
                             s["lens"], scale, pages=s["pages"])
        return s["y"]
    if case["op"] == "norm_rope":
        return (plain_norm_rope(s, s["q"], s["q_weight"]), plain_norm_rope(s, s["k"], s["k_weight"]))
    return plain_packed(s, scale) if case["op"] == "packed" else plain_prefix(s, scale)


def plain_norm_rope(s, x, weight):
    case = s["case"]
    rot, half = case["rot"], case["rot"] // 2
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    pos = s["positions"].long().view(case["axes"], -1)
    at = pos[s["axis"]].T  # [tokens, half]: the position that turns each pair
    pair = torch.arange(half, device=x.device)
    cos, sin = s["table"][at, pair][:, None], s["table"][at, half + pair][:, None]
    if case["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., rot:]], dim=-1).to(x.dtype)


def weighted(scores, seen):
    """exp(scores - row maximum) where `seen`, 0 elsewhere, and the row sums (1 for rows that see nothing)."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1)
    return p, torch.where(total == 0, torch.ones_like(total), total)


def plain_packed(s, scale):
    case, q, k = s["case"], s["q"], s["k"]
    t, n = q.shape[0], k.shape[0]
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    row, key = torch.arange(t, device=q.device), torch.arange(n, device=q.device)
    mine, of = torch.bucketize(row, qs[1:], right=True), torch.bucketize(key, ks[1:], right=True)
    inside = mine < case["seqs"]  # rows behind the last sequence are left as they were
    seen = (mine[:, None] == of) & inside[:, None]
    if case["causal"]:  # the last query of a sequence sees its last key
        m = mine.clamp(max=case["seqs"] - 1)
        seen = seen & (key - ks[1:][m][:, None] <= (row - qs[1:][m])[:, None])
    qf = q.float().view(t, case["kv_heads"], -1, case["d"])
    p, total = weighted(torch.einsum("tkgd,skd->kgts", qf, k.float()) * scale, seen)
    o = torch.einsum("kgts,skd->tkgd", p, s["v"].float()) / total.permute(2, 0, 1)[..., None]
    return torch.where(inside[:, None, None], o.reshape(q.shape).to(q.dtype), s["y"])


def plain_prefix(s, scale):
    case, q = s["case"], s["q"]
    b, t = q.shape[:2]
    page = s["k_pages"].shape[1]
    wide = s["k_pages"].shape[0] // b
    table = s["pages"].long() if s["pages"] is not None else \
        torch.arange(b, device=q.device)[:, None]
    j = torch.arange(wide * page, device=q.device)
    rows = table[:, j // page] * page + j % page
    k = s["k_pages"].flatten(0, 1)[rows].float()
    v = s["v_pages"].flatten(0, 1)[rows].float()
    qf = q.float().view(b, t, case["kv_heads"], -1, case["d"])
    front = torch.einsum("btkgd,skd->bkgts", qf, s["prefix_k"].float()) * scale
    back = torch.einsum("btkgd,bskd->bkgts", qf, k) * scale
    step = torch.arange(t, device=q.device)
    seen = j <= (s["lens"].long()[:, None] - t + step)[..., None]  # [batch, steps, keys]
    seen = torch.cat([torch.ones(b, t, case["prefix"], dtype=torch.bool, device=q.device), seen], dim=-1)
    p, total = weighted(torch.cat([front, back], dim=-1), seen[:, None, None])
    o = torch.einsum("bkgts,skd->btkgd", p[..., :case["prefix"]], s["prefix_v"].float()) + \
        torch.einsum("bkgts,bskd->btkgd", p[..., case["prefix"]:], v)
    return (o / total.permute(0, 3, 1, 2)[..., None]).reshape(q.shape).to(q.dtype)


# ---- 64 bits ------------------------------------------------------------------

def exact(case, seed):
    """The same from the definitions in 64 bits, one sequence or request and one head at a time."""
    s = prepare(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["d"]

    def attend(q, k, v, seen):
        z = (q @ k.T) * d ** -0.5
        z[~seen] = -math.inf
        w = torch.softmax(z, dim=-1)
        w[~seen.any(-1)] = 0
        return w @ v

    if case["op"] == "norm_rope":
        return tuple(exact_norm_rope(case, s, s[n], s[n + "_weight"]) for n in "qk")
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "packed":
        q0 = k0 = 0
        for nq, nk in zip(*packed_lengths(case)):
            i, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
            seen = j[None] <= i[:, None] + (nk - nq) if case["causal"] else \
                torch.ones(nq, nk, dtype=torch.bool, device="cuda")
            for head in range(h):
                c = head // (h // kv)
                y[q0:q0 + nq, head] = attend(s["q"][q0:q0 + nq, head].double(),
                                             s["k"][k0:k0 + nk, c].double(),
                                             s["v"][k0:k0 + nk, c].double(), seen)
            q0, k0 = q0 + nq, k0 + nk
        return y
    t, page = case["steps"], s["k_pages"].shape[1]
    front = torch.stack([s["prefix_k"], s["prefix_v"]]).double()
    for r, n in enumerate(prefix_lengths(case)):
        have = s["pages"][r].tolist() if s["pages"] is not None else [r]
        tail = torch.stack([torch.cat([x[p] for p in have[:-(-n // page)]])[:n]
                            for x in (s["k_pages"], s["v_pages"])]).double()
        keys, values = torch.cat([front, tail], dim=1)
        at = torch.arange(keys.shape[0], device="cuda")
        seen = at[None] < case["prefix"] + n - t + 1 + torch.arange(t, device="cuda")[:, None]
        for c in range(kv):  # the heads of a group see the same keys
            g = h // kv
            q = s["q"][r, :, c * g:(c + 1) * g].double().reshape(t * g, d)
            y[r, :, c * g:(c + 1) * g] = attend(q, keys[:, c], values[:, c],
                                                seen.repeat_interleave(g, 0)).view(t, g, d)
    return y


def exact_norm_rope(case, s, x, weight):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + 1e-6) * weight.double()
    half = case["rot"] // 2
    y = x.clone()
    pos = s["positions"].view(case["axes"], -1)
    i = 0
    for axis, count in enumerate(s["sections"]):
        for i in range(i, i + count):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            row = s["table"][pos[axis].long()].double()
            c, z = row[:, i, None], row[:, half + i, None]
            y[..., a] = x[..., a] * c - x[..., b] * z
            y[..., b] = x[..., b] * c + x[..., a] * z
        i += 1
    return y
