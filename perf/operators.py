"""Cases of the token-generation operators: rotary positions, appending to a
paged key-value cache, attention of one new token over that cache, and products
with 4-bit weights.

`run` computes them in plain torch operations, or, where `own` is true, through
pyflame_b200's public calls.  Every size is either this repository's own (the
encoder's 12 heads of 64, the Linear chain's 4096 and 16384) or generic.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # queries of two 4096-token prompts, rotated before attention
        dict(name="rope prompt bf16", op="rope", dtype="bf16", batch=2, seq=4096, heads=32, dim=128, rot=128,
             layout="half", scaling="none", backward=False),
        # gradients of a training step through a partly rotated head, the encoder's 12 heads of 64
        dict(name="rope gradient fp32", op="rope", dtype="fp32", batch=1, seq=2047, heads=12, dim=64, rot=32,
             layout="interleaved", scaling="linear", backward=True),
        # one user, one token: the smallest call of a decoder layer
        dict(name="append token fp32", op="append", dtype="fp32", tokens=1, heads=12, kv_heads=12, dim=64, rot=64,
             layout="half", scaling="none", page=16, skip=0),
        # a long prompt entering the cache, its rotation scaled for a context eight times the trained one
        dict(name="append prompt fp16", op="append", dtype="fp16", tokens=8191, heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", scaling="yarn", page=16, skip=0),
        # one user with a short context, statistics returned for joining with another part of it
        dict(name="attend short fp32", op="attend", dtype="fp32", batch=1, longest=333, shortest=333, heads=12,
             kv_heads=12, dim=64, page=16, window=0, lse=True),
        # one user with a long document
        dict(name="attend long bf16", op="attend", dtype="bf16", batch=1, longest=131071, shortest=131071, heads=64,
             kv_heads=8, dim=128, page=64, window=0, lse=False),
        # a batch in the middle of serving: every length, empty rows of a padded batch among them
        dict(name="attend ragged fp16", op="attend", dtype="fp16", batch=48, longest=8192, shortest=0, heads=32,
             kv_heads=8, dim=128, page=16, window=0, lse=False),
        # the largest: a full machine
        dict(name="attend full bf16", op="attend", dtype="bf16", batch=128, longest=8192, shortest=2048, heads=32,
             kv_heads=8, dim=128, page=32, window=0, lse=False),
        # every head its own keys, an uncommon head size and page, a sliding window
        dict(name="attend window fp32", op="attend", dtype="fp32", batch=7, longest=5000, shortest=1, heads=20,
             kv_heads=20, dim=80, page=13, window=1000, lse=True),
        # one token through a square projection
        dict(name="linear4 token bf16", op="linear4", dtype="bf16", rows=1, inner=4096, outer=4096, group=128,
             zeros=False, bias=False),
        # one token through the Linear chain's first layer, in this framework's own type
        dict(name="linear4 up fp32", op="linear4", dtype="fp32", rows=1, inner=4096, outer=16384, group=64,
             zeros=True, bias=True),
        # a batch of tokens through its second layer, the finest groups
        dict(name="linear4 rows fp16", op="linear4", dtype="fp16", rows=33, inner=16384, outer=4096, group=32,
             zeros=True, bias=False),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "linear4"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "linear4":
        rows = _log(rng, 1, 40)
        inner, outer = _log(rng, 60, 16384), _log(rng, 60, 16384)
        return dict(op=op, dtype=dtype, rows=rows, inner=inner, outer=outer, group=rng.choice([32, 64, 128]),
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
    dim = rng.choice([64, 72, 80, 96, 128, 128])
    rot = rng.choice([dim, dim, dim // 2])
    turn = dict(rot=rot, layout=rng.choice(["half", "interleaved"]),
                scaling=rng.choice(["none", "linear", "ntk", "yarn"]))
    if op == "rope":
        heads = rng.choice([1, 5, 12, 32])
        return dict(op=op, dtype=dtype, batch=rng.choice([1, 2, 3]), seq=_log(rng, 1, 5000), heads=heads, dim=dim,
                    backward=rng.random() < 0.5, **turn)
    kv_heads = rng.choice([1, 2, 3, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "append":
        tokens = _log(rng, 1, 6000)
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([1, 7, 16, 32, 64]), skip=tokens // 9, **turn)
    batch = _log(rng, 1, 64)
    # at most a quarter of the largest listed case's cache
    most = max(8, min(60000, int(1.5e8 // (batch * kv_heads * dim))))
    longest = _log(rng, 1, most)
    return dict(op=op, dtype=dtype, batch=batch, longest=longest, shortest=rng.randint(0, longest), heads=heads,
                kv_heads=kv_heads, dim=dim, page=rng.choice([1, 7, 13, 16, 32, 64]),
                window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]), lse=rng.random() < 0.3)


def lengths(case):
    """The sequences' lengths: fixed by the case, so that its work is; the seed orders them."""
    n, low, high = case["batch"], case["shortest"], case["longest"]
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def angles(case):
    """inverse frequencies of a case's rotation in 64 bits, and the factor on its cosines and sines."""
    r, base, factor, trained = case["rot"], 10000.0, 8.0, 4096
    i = torch.arange(r // 2, dtype=torch.float64)
    if case["scaling"] == "ntk":
        base = base * factor ** (r / (r - 2))
    inv = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        inv = inv / factor
    if case["scaling"] == "yarn":
        low, high = (r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
    return inv, 0.1 * math.log(factor) + 1 if case["scaling"] == "yarn" else 1.0


def _rotary(case):
    """The framework's rotation of a case."""
    import pyflame_b200 as pf
    kind = case["scaling"]
    scaling = None if kind == "none" else {"type": kind, "factor": 8.0}
    if kind == "yarn":
        scaling["original_max_position"] = 4096
    return pf.RotaryEmbedding(case["dim"], case["rot"], layout=case["layout"], scaling=scaling, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=t)

    if op == "linear4":
        n, k, group = case["outer"], case["inner"], case["group"]
        s = {"x": normal(case["rows"], k),
             # two values a byte, the even column in the low half
             "packed": torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8),
             "scales": ((torch.rand((n, -(-k // group)), generator=g, device="cuda") + 0.5) / (6 * k ** 0.5)).half(),
             "zeros": None, "bias": normal(n) if case["bias"] else None, "inner": k, "group": group}
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 12, (n, -(-k // group)), generator=g, device="cuda", dtype=torch.uint8)
        if own:
            import pyflame_b200 as pf
            s["layer"] = pf.Linear4bit(s["packed"], s["scales"], s["zeros"], s["bias"], in_features=k, group_size=group)
        return {"op": op, "t": t, **s}
    if op == "rope":
        inv, factor = angles(case)
        s = {"x": normal(case["batch"], case["seq"], case["heads"], case["dim"]),
             "positions": torch.arange(case["seq"], device="cuda") + int(torch.randint(0, 100000, (), generator=g, device="cuda")),
             "inv": inv.cuda(), "factor": factor, "case": case, "rotary": _rotary(case) if own else None}
        return {"op": op, "t": t, **s}
    if op == "append":
        inv, factor = angles(case)
        n, h, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        qkv = normal(n, (h + 2 * hk) * d)  # one projection's output, of which q, k and v are slices
        pages = -(-n // page) + 5
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
        if case["skip"]:  # rows of padding
            slots[torch.randperm(n, generator=g, device="cuda")[:case["skip"]]] = -1
        s = {"q": qkv[:, :h * d].view(n, h, d), "k": qkv[:, h * d:(h + hk) * d].view(n, hk, d),
             "v": qkv[:, (h + hk) * d:].view(n, hk, d), "q_out": torch.zeros(n, h, d, device="cuda", dtype=t),
             "slots": slots, "positions": torch.randint(0, 32768, (n,), generator=g, device="cuda"),
             "k_cache": normal(pages, page, hk, d), "v_cache": normal(pages, page, hk, d),
             "inv": inv.cuda(), "factor": factor, "case": case}
        if own:
            import pyflame_b200 as pf
            s["cache"], s["rotary"] = pf.PagedKVCache.from_tensors(s["k_cache"], s["v_cache"]), _rotary(case)
        return {"op": op, "t": t, **s}
    lens, page = lengths(case), case["page"]
    order = torch.randperm(len(lens), generator=g, device="cuda").tolist()
    lens = [lens[i] for i in order]
    need = [-(-n // page) for n in lens]
    pages, most = sum(need) + 3, max(1, max(need))
    table = torch.zeros(len(lens), most, dtype=torch.int32)
    at, free = 0, torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    for b, n in enumerate(need):
        table[b, :n] = free[at:at + n]
        at += n
    s = {"q": normal(case["batch"], case["heads"], case["dim"]),
         "k_cache": normal(pages, page, case["kv_heads"], case["dim"]),
         "v_cache": normal(pages, page, case["kv_heads"], case["dim"]),
         "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "window": case["window"], "lse": case["lse"]}
    if own:
        import pyflame_b200 as pf
        s["cache"] = pf.PagedKVCache.from_tensors(s["k_cache"], s["v_cache"])
    return {"op": op, "t": t, **s}


def _rotate(x, positions, inv, factor, case, sign=1.0):
    """x [..., tokens, heads, dim] rotated in 32 bits by angles taken in 64."""
    a = positions.double()[:, None] * inv
    c, s = ((f(a) * factor).float()[:, None, :] for f in (torch.cos, torch.sin))
    s, r, x = s * sign, case["rot"], x.float()
    y = x.clone()
    if case["layout"] == "half":
        i, j = slice(0, r // 2), slice(r // 2, r)
    else:
        i, j = slice(0, r, 2), slice(1, r, 2)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def run(s):
    op, t = s["op"], s["t"]
    if own:
        if op == "linear4":
            return s["layer"](s["x"])
        if op == "rope":
            turn = s["rotary"].backward if s["case"]["backward"] else s["rotary"].apply
            return turn(s["x"], s["positions"])
        if op == "append":
            s["cache"].append(s["k"], s["v"], s["slots"], positions=s["positions"], rotary=s["rotary"], q=s["q"],
                              q_out=s["q_out"])
            return s["k_cache"], s["v_cache"], s["q_out"]
        return s["cache"].attend(s["q"], s["table"], s["lens"], window=s["window"], return_lse=s["lse"])
    if op == "linear4":
        k, group = s["inner"], s["group"]
        q = torch.stack((s["packed"] & 15, s["packed"] >> 4), -1).flatten(1)[:, :k].float()
        z = s["zeros"].float() if s["zeros"] is not None else torch.full_like(s["scales"], 8, dtype=torch.float32)
        scales = s["scales"].float().repeat_interleave(group, 1)[:, :k]
        y = s["x"].float() @ ((q - z.repeat_interleave(group, 1)[:, :k]) * scales).T
        return (y if s["bias"] is None else y + s["bias"].float()).to(t)
    if op == "rope":
        sign = -1.0 if s["case"]["backward"] else 1.0
        return _rotate(s["x"], s["positions"], s["inv"], s["factor"], s["case"], sign).to(t)
    if op == "append":
        keep = s["slots"] >= 0
        at = s["slots"][keep]
        s["k_cache"].flatten(0, 1)[at] = _rotate(s["k"], s["positions"], s["inv"], s["factor"], s["case"]).to(t)[keep]
        s["v_cache"].flatten(0, 1)[at] = s["v"][keep]
        s["q_out"][keep] = _rotate(s["q"], s["positions"], s["inv"], s["factor"], s["case"]).to(t)[keep]
        return s["k_cache"], s["v_cache"], s["q_out"]
    q, lens = s["q"].float(), s["lens"].long()
    b, h, d = q.shape
    k, v = (c[s["table"].long()].flatten(1, 2).float() for c in (s["k_cache"], s["v_cache"]))  # [b, keys, kv heads, d]
    hk = k.shape[2]
    j = torch.arange(k.shape[1], device="cuda")
    seen = j < lens[:, None]
    if s["window"]:
        seen = seen & (j >= lens[:, None] - s["window"])
    score = torch.einsum("bghd,bkgd->bghk", q.view(b, hk, h // hk, d), k) / math.sqrt(d)
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bghk,bkgd->bghd", p, v) / total.clamp(min=1e-30)
    if s["lse"]:
        return o.reshape(b, h, d).to(t), (top + total.log()).reshape(b, h)
    return o.reshape(b, h, d).to(t)


def work(case):
    e, op = SIZE[case["dtype"]], case["op"]
    if op == "linear4":
        m, n, k = case["rows"], case["outer"], case["inner"]
        groups = n * -(-k // case["group"])
        return {"bytes": n * k // 2 + groups * (3 if case["zeros"] else 2) + e * m * (n + k) + (e * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if op == "rope":
        x = case["batch"] * case["seq"] * case["heads"]
        return {"bytes": 2 * e * x * case["dim"] + 8 * case["seq"], "flops": 3.0 * x * case["rot"]}
    if op == "append":
        n, h, hk, d = case["tokens"] - case["skip"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": 2 * e * n * (h + 2 * hk) * d + 16 * case["tokens"], "flops": 3.0 * n * (h + hk) * case["rot"]}
    lens = [min(n, case["window"] or n) for n in lengths(case)]
    b, h, hk, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    return {"bytes": 2 * e * sum(lens) * hk * d + 2 * e * b * h * d + 4 * b + sum(4 * -(-n // page) for n in lens)
            + (4 * b * h if case["lse"] else 0), "flops": 4.0 * sum(lens) * h * d}


def _turned(x, positions, case, way=1):
    """x rotated in 64 bits as complex numbers."""
    inv, factor = angles(case)
    r = case["rot"]
    x = x.double()
    pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else x[..., :r].unflatten(-1, (r // 2, 2))
    z = torch.view_as_complex(pairs.contiguous())
    a = way * torch.outer(positions.double(), inv.to(positions.device))
    z = torch.view_as_real(z * torch.polar(torch.full_like(a, factor), a)[:, None])
    z = z.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else z.flatten(-2)
    return torch.cat((z, x[..., r:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _turned(s["x"], s["positions"], case, -1 if case["backward"] else 1)
    if op == "append":
        k, v, q = s["k_cache"].double(), s["v_cache"].double(), s["q_out"].double()
        kr, qr = (_turned(s[n], s["positions"], case) for n in ("k", "q"))
        page = case["page"]
        live = [(i, p) for i, p in enumerate(s["slots"].tolist()) if p >= 0]
        if live:
            i, p = (torch.tensor(x, device="cuda") for x in zip(*live))
            k[p // page, p % page], v[p // page, p % page], q[i] = kr[i], s["v"][i].double(), qr[i]
        return k, v, q
    if op == "linear4":
        k, group = case["inner"], case["group"]
        x, y = s["x"].double(), torch.zeros(case["rows"], case["outer"], dtype=torch.float64, device="cuda")
        for lo in range(0, k, group):  # a group of columns at a time
            c = torch.arange(lo, min(k, lo + group), device="cuda")
            q = (s["packed"][:, c // 2].int() >> (4 * (c % 2)).int()) & 15
            z = s["zeros"][:, lo // group].double()[:, None] if case["zeros"] else 8.0
            y += x[:, c] @ ((q.double() - z) * s["scales"][:, lo // group].double()[:, None]).T
        return y if s["bias"] is None else y + s["bias"].double()
    out = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    each, page = case["heads"] // case["kv_heads"], case["page"]
    for b, n in enumerate(s["lens"].tolist()):
        j = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        if not n:
            continue
        at = s["table"][b, j // page].long()
        k, v = (s[c][at, j % page].double().transpose(0, 1) for c in ("k_cache", "v_cache"))  # [kv heads, keys, dim]
        score = s["q"][b].double().view(case["kv_heads"], each, -1) @ k.transpose(1, 2) * case["dim"] ** -0.5
        lse[b] = torch.logsumexp(score, -1).flatten()
        out[b] = (torch.softmax(score, -1) @ v).flatten(0, 1)
    return (out, lse) if case["lse"] else out
