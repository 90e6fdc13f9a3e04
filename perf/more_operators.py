"""Cases of the operators of a serving decoder layer: a paged key-value cache
in 4 bits (appending to it, attention of one new token over it), low-rank
adapters of many requests beside a shared projection, and a mixture-of-experts
layer for a few tokens.

`run` computes them in plain torch operations, or, where `own` is true, through
pyflame_b200's public calls.  Every size is either this repository's own (the
encoder's 12 heads of 64 and width 768, the Linear chain's 4096 and 16384) or
generic.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # one user, one token: the smallest call of a decoder layer; what was stored is read back
        dict(name="append4 token fp32", op="append4", dtype="fp32", tokens=1, heads=12, kv_heads=12, dim=64, group=32, rot=64,
             layout="half", scaling="none", page=16, skip=0),
        # a long prompt entering the cache, its rotation scaled for a context eight times the trained one
        dict(name="append4 prompt fp16", op="append4", dtype="fp16", tokens=8191, heads=32, kv_heads=8, dim=128, group=64,
             rot=128, layout="half", scaling="yarn", page=16, skip=0),
        # one user with a short context: every head its own keys, an uncommon head size and page, a sliding window,
        # statistics returned for joining with another part of the context
        dict(name="attend4 short fp32", op="attend4", dtype="fp32", batch=1, longest=333, shortest=333, heads=20, kv_heads=20,
             dim=80, group=64, page=13, window=250, lse=True),
        # one user with a long document
        dict(name="attend4 long bf16", op="attend4", dtype="bf16", batch=1, longest=131071, shortest=131071, heads=64,
             kv_heads=8, dim=128, group=64, page=64, window=0, lse=False),
        # a batch in the middle of serving: every length, empty rows of a padded batch among them; the finest groups
        dict(name="attend4 ragged fp16", op="attend4", dtype="fp16", batch=48, longest=8192, shortest=0, heads=32, kv_heads=8,
             dim=128, group=32, page=16, window=0, lse=False),
        # a full machine
        dict(name="attend4 full bf16", op="attend4", dtype="bf16", batch=128, longest=8192, shortest=2048, heads=32,
             kv_heads=8, dim=128, group=64, page=32, window=0, lse=False),
        # one user's token through a square projection with its adapter
        dict(name="adapters token bf16", op="adapters", dtype="bf16", rows=1, inner=4096, outer=4096, rank=16, adapters=8,
             order="each", skip=0),
        # a batch of tokens, every one of another user, some without an adapter, through the Linear chain's first layer
        dict(name="adapters batch fp16", op="adapters", dtype="fp16", rows=61, inner=4096, outer=16384, rank=64, adapters=64,
             order="each", skip=6),
        # prompts of five users, one behind the other
        dict(name="adapters prompts bf16", op="adapters", dtype="bf16", rows=8191, inner=4096, outer=4096, rank=16, adapters=5,
             order="runs", skip=0),
        # one token through many small experts
        dict(name="experts token bf16", op="experts", dtype="bf16", tokens=1, experts=64, top=6, width=2048, inner=1408,
             renormalize=False, activation="silu"),
        # a few tokens through few experts, in this framework's own type
        dict(name="experts few fp32", op="experts", dtype="fp32", tokens=5, experts=8, top=2, width=768, inner=2048,
             renormalize=True, activation="gelu"),
        # the largest: a batch of tokens that needs nearly every expert
        dict(name="experts batch fp16", op="experts", dtype="fp16", tokens=64, experts=128, top=8, width=2048, inner=768,
             renormalize=True, activation="silu"),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append4", "attend4", "attend4", "adapters", "adapters", "experts", "experts"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "experts":
        experts = rng.choice([1, 4, 8, 16, 60, 64, 128])
        width, inner = _log(rng, 60, 4096), _log(rng, 30, 4096)
        most = 3e8 / experts / 3  # weights of an expert's matrix
        while width * inner > most:
            width, inner = width * 3 // 4, inner * 3 // 4
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 64), experts=experts, top=rng.randint(1, min(8, experts)),
                    width=width, inner=inner, renormalize=rng.random() < 0.5, activation=rng.choice(["silu", "gelu"]))
    if op == "adapters":
        inner, outer, rank = _log(rng, 60, 8192), _log(rng, 60, 8192), rng.choice([4, 8, 16, 17, 32, 64])
        adapters = rng.choice([1, 2, 5, 16, 64])
        # at most the listed prompts' values and products
        most = min(2.5e7 / (inner + outer), 5e12 / ((inner + outer) * rank * adapters * 10))
        rows = _log(rng, 1, max(8, int(most)))
        return dict(op=op, dtype=dtype, rows=rows, inner=inner, outer=outer, rank=rank, adapters=adapters,
                    order=rng.choice(["each", "runs"]), skip=rng.choice([0, rows // 9]))
    dim, group = rng.choice([64, 72, 80, 96, 128, 128]), rng.choice([32, 64, 128])
    if op == "append4":
        kv_heads = rng.choice([1, 2, 3, 8, 12])
        tokens = _log(rng, 1, 6000)
        return dict(op=op, dtype=dtype, tokens=tokens, heads=kv_heads * rng.choice([1, 2, 3, 4]), kv_heads=kv_heads, dim=dim,
                    group=group, rot=rng.choice([dim, dim, dim // 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), page=rng.choice([1, 7, 16, 32, 64]), skip=tokens // 9)
    batch = _log(rng, 1, 64)
    kv_heads = rng.choice([1, 2, 3, 8, 12])
    # at most a quarter of the largest listed attention's cache
    most = max(8, min(120000, int(1.7e8 // (batch * kv_heads * dim))))
    longest = _log(rng, 1, most)
    return dict(op=op, dtype=dtype, batch=batch, longest=longest, shortest=rng.randint(0, longest),
                heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv_heads, dim=dim, group=group,
                page=rng.choice([1, 7, 13, 16, 32, 64]), window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]),
                lse=rng.random() < 0.3)


def lengths(case):
    """The sequences' lengths: fixed by the case, so that its work is; the seed orders them."""
    n, low, high = case["batch"], case["shortest"], case["longest"]
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def owners(case):
    """The rows' adapters, as often as the case says; -1: none.  The seed orders those of separate requests."""
    n, a, live = case["rows"], case["adapters"], case["rows"] - case["skip"]
    if case["order"] == "runs":  # runs of unlike lengths, the rows without one in the middle
        cuts = [live * (i + 1) * (i + 2) // (a * (a + 1)) for i in range(a)]
        own_of = [next(i for i in range(a) if r < cuts[i]) for r in range(live)]
        return own_of[:live // 2] + [-1] * case["skip"] + own_of[live // 2:]
    return [i % a for i in range(live)] + [-1] * (n - live)


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


def _quantize(x, group):
    """x [..., dim] in float32 as (codes 0 to 15, steps, lows): each group of values in 16 even steps from its least value
    on, steps and lows in bfloat16.  32-bit operations one at a time: which code a value gets is a decision."""
    d = x.shape[-1]
    n = -(-d // group)
    if n * group != d:  # the last group is shorter: filled up with its last value, which changes neither end
        x = torch.cat((x, x[..., -1:].expand(*x.shape[:-1], n * group - d)), -1)
    x = x.unflatten(-1, (n, group))
    low = x.amin(-1).bfloat16().float()
    step = ((x.amax(-1) - low) / 15).bfloat16().float()
    step = torch.where(step < 2.0 ** -126, 0.0, step)
    times = torch.where(step > 0, 1 / step, 0.0)
    codes = ((x - low[..., None]) * times[..., None]).round().clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2)[..., :d], step, low


def _values(codes, step, low, group):
    d = codes.shape[-1]
    step, low = (s.float().repeat_interleave(group, -1)[..., :d] for s in (step, low))
    return codes.float() * step + low


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=t)

    if op == "experts":
        n, e, d, f = case["tokens"], case["experts"], case["width"], case["inner"]
        s = {"x": normal(n, d), "router": normal(e, d) / d ** 0.5, "gate_up": normal(e, 2 * f, d).div_(d ** 0.5),
             "down": normal(e, d, f).div_(f ** 0.5), "case": case}
        if own:
            import pyflame_b200 as pf
            s["layer"] = pf.MixtureOfExperts(s["router"], s["gate_up"], s["down"], case["top"],
                                             renormalize=case["renormalize"], activation=case["activation"])
        return {"op": op, "t": t, **s}
    if op == "adapters":
        n, a, r, k, m = case["rows"], case["adapters"], case["rank"], case["inner"], case["outer"]
        index = torch.tensor(owners(case), dtype=torch.int32, device="cuda")
        if case["order"] == "each":
            index = index[torch.randperm(n, generator=g, device="cuda")]
        s = {"x": normal(n, k), "base": normal(n, m), "index": index, "a": normal(a, r, k) / k ** 0.5, "b": normal(a, m, r),
             "scales": torch.rand(a, generator=g, device="cuda") + 0.5}
        if own:
            import pyflame_b200 as pf
            s["layer"] = pf.LowRankAdapters(a, k, m, r, dtype=t)
            for i, scale in enumerate(s["scales"].tolist()):
                s["layer"].load(i, s["a"][i], s["b"][i], scale)
        return {"op": op, "t": t, **s}
    if op == "append4":
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
             "inv": inv.cuda(), "factor": factor, "case": case}
        if own:
            import pyflame_b200 as pf
            s["cache"] = pf.PagedKVCache4bit(pages, page, hk, d, group_size=case["group"])
            s["rotary"] = _rotary(case)
        else:  # of keys and of values: two codes a byte, the even value in the low half; steps and lows
            shape, groups = (pages * page, hk), -(-d // case["group"])
            s["stored"] = [(torch.zeros(*shape, d // 2, device="cuda", dtype=torch.uint8),
                            *(torch.zeros(*shape, groups, device="cuda", dtype=torch.bfloat16) for _ in range(2)))
                           for _ in range(2)]
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
    hk, d = case["kv_heads"], case["dim"]
    k, v = (normal(pages * page, hk, d) for _ in range(2))
    # some channels of keys stand far from the others and from 0
    k += 4 * (torch.rand(hk, d, generator=g, device="cuda") < 0.05).to(t)
    s = {"q": normal(case["batch"], case["heads"], d), "table": table.cuda(),
         "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "window": case["window"], "lse": case["lse"], "case": case}
    if own:
        import pyflame_b200 as pf
        s["cache"] = pf.PagedKVCache4bit(pages, page, hk, d, group_size=case["group"])
        s["cache"].append(k, v, torch.arange(pages * page, device="cuda"))
    else:
        s["stored"] = []
        for x in (k, v):
            parts = []
            for some in x.split(65536):  # the codes of many tokens at once would take room
                codes, step, low = _quantize(some.float(), case["group"])
                parts.append((codes[..., 0::2] | codes[..., 1::2] << 4, step.bfloat16(), low.bfloat16()))
            s["stored"].append(tuple(torch.cat(p).unflatten(0, (pages, page)) for p in zip(*parts)))
    return {"op": op, "t": t, **s}


def _rotate(x, positions, inv, factor, case):
    """x [tokens, heads, dim] rotated in 64 bits: the code that a value gets is a decision."""
    a = positions.double()[:, None] * inv
    c, s = ((f(a) * factor)[:, None, :] for f in (torch.cos, torch.sin))
    r, x = case["rot"], x.double()
    y = x.clone()
    if case["layout"] == "half":
        i, j = slice(0, r // 2), slice(r // 2, r)
    else:
        i, j = slice(0, r, 2), slice(1, r, 2)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _plain_experts(s):
    case, t, x = s["case"], s["t"], s["x"].float()
    logits = s["x"].double() @ s["router"].double().T  # in 64 bits: which experts a token takes is a decision
    order = torch.sort(logits, descending=True, stable=True)
    chosen, top = order.indices[:, :case["top"]], order.values[:, :case["top"]]
    best = logits.amax(-1, keepdim=True)
    part = (top - best).exp()
    part = part / (part if case["renormalize"] else (logits - best).exp()).sum(-1, keepdim=True)
    part = part.float()
    f = case["inner"]

    def act(gate):
        if case["activation"] == "silu":
            return gate / (1 + (-gate).exp())
        return 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))

    if chosen.numel() < case["experts"]:  # the chosen experts' matrices for every token
        both = (s["gate_up"][chosen].float() @ x[:, None, :, None])[..., 0]
        h = act(both[..., :f]) * both[..., f:] * part[..., None]
        return (s["down"][chosen].float() @ h[..., None])[..., 0].sum(1).to(t), chosen.int(), part
    y = torch.zeros_like(x)
    for e in range(case["experts"]):  # every expert for all tokens
        share = (part * (chosen == e)).sum(-1, keepdim=True)
        both = x @ s["gate_up"][e].float().T
        y += share * ((act(both[:, :f]) * both[:, f:]) @ s["down"][e].float().T)
    return y.to(t), chosen.int(), part


def run(s):
    op, t = s["op"], s["t"]
    if own:
        if op == "experts":
            return s["layer"](s["x"], return_routing=True)
        if op == "adapters":
            return s["layer"](s["x"], s["index"], s["base"])
        if op == "append4":
            s["cache"].append(s["k"], s["v"], s["slots"], positions=s["positions"], rotary=s["rotary"], q=s["q"],
                              q_out=s["q_out"])
            return *s["cache"].read(s["slots"], t), s["q_out"]
        return s["cache"].attend(s["q"], s["table"], s["lens"], window=s["window"], return_lse=s["lse"])
    if op == "experts":
        return _plain_experts(s)
    if op == "adapters":
        x, index, a, b = s["x"].float(), s["index"].long(), s["a"], s["b"]
        scale = torch.where(index >= 0, s["scales"][index.clamp(min=0)], 0.0)[:, None]
        if len(x) <= len(a):  # every row's own matrices
            at = index.clamp(min=0)
            h = (a[at].float() @ x[:, :, None]) * scale[:, :, None]
            add = (b[at].float() @ h)[:, :, 0]
        else:  # products with all adapters, of which each row keeps its own
            h = (x @ a.flatten(0, 1).float().T).unflatten(-1, a.shape[:2])
            h = h * (scale * (index[:, None] == torch.arange(len(a), device="cuda")))[:, :, None]
            add = h.flatten(1) @ b.transpose(1, 2).flatten(0, 1).float()
        return (s["base"].float() + add).to(t)
    case = s["case"]
    group = case["group"]
    if op == "append4":
        keep = s["slots"] >= 0
        at = s["slots"][keep]
        turn = s["positions"], s["inv"], s["factor"], case
        back = []
        for x, (codes, step, low) in zip((_rotate(s["k"], *turn).float(), s["v"].float()), s["stored"]):
            c, st, lo = _quantize(x[keep], group)
            codes[at], step[at], low[at] = c[..., 0::2] | c[..., 1::2] << 4, st.bfloat16(), lo.bfloat16()
            at0 = s["slots"].clamp(min=0)
            back.append((_values(_unpack(codes[at0]), step[at0], low[at0], group) * keep[:, None, None]).to(t))
        s["q_out"][keep] = _rotate(s["q"], *turn)[keep].to(t)
        return *back, s["q_out"]
    q, lens = s["q"].float(), s["lens"].long()
    b, h, d = q.shape
    table = s["table"].long()
    k, v = (_values(_unpack(c[table]).flatten(1, 2), st[table].flatten(1, 2), lo[table].flatten(1, 2), group)
            for c, st, lo in s["stored"])  # [b, keys, kv heads, d]
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
    if op == "experts":
        n, k, d, f = case["tokens"], case["top"], case["width"], case["inner"]
        used = case["experts"] * (1 - (1 - k / case["experts"]) ** n)  # as many as independent choices leave in use
        return {"bytes": int(3 * e * d * f * used) + e * (case["experts"] * d + 2 * n * d) + 8 * n * k,
                "flops": 6.0 * n * k * d * f + 2.0 * n * case["experts"] * d}
    if op == "adapters":
        n, r, k, m = case["rows"], case["rank"], case["inner"], case["outer"]
        used = len(set(owners(case)) - {-1})
        live = n - case["skip"]
        return {"bytes": e * (live * k + 2 * n * m + used * r * (k + m)) + 4 * (n + used), "flops": 2.0 * live * r * (k + m)}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    token = hk * (d + 8 * -(-d // case["group"]))  # bytes of a token in the cache
    if op == "append4":
        n = case["tokens"] - case["skip"]
        return {"bytes": 2 * e * n * (h + 2 * hk) * d + 2 * n * token + 24 * case["tokens"],
                "flops": 3.0 * n * (h + hk) * case["rot"] + 10.0 * n * hk * d}
    lens = [min(n, case["window"] or n) for n in lengths(case)]
    b, page = case["batch"], case["page"]
    return {"bytes": sum(lens) * token + 2 * e * b * h * d + 4 * b + sum(4 * -(-n // page) for n in lens)
            + (4 * b * h if case["lse"] else 0), "flops": 4.0 * sum(lens) * h * d}


def _turned(x, positions, case):
    """x rotated in 64 bits as complex numbers."""
    inv, factor = angles(case)
    r = case["rot"]
    x = x.double()
    pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else x[..., :r].unflatten(-1, (r // 2, 2))
    z = torch.view_as_complex(pairs.contiguous())
    a = torch.outer(positions.double(), inv.to(positions.device))
    z = torch.view_as_real(z * torch.polar(torch.full_like(a, factor), a)[:, None])
    z = z.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else z.flatten(-2)
    return torch.cat((z, x[..., r:]), -1)


def _kept(x, group):
    """The values that the 4-bit cache keeps of x [..., dim], a group at a time, in 64 bits from 32-bit values."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[-1], group):
        part = x[..., at:at + group].float()
        least, most = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
        least = least.to(torch.bfloat16).float()
        width = torch.div(most - least, 15.0).to(torch.bfloat16).float()
        width[width < torch.finfo(torch.float32).tiny] = 0
        inverse = torch.where(width == 0, torch.zeros_like(width), width.reciprocal())
        code = torch.round((part - least).mul(inverse)).clamp(max=15).clamp(min=0)
        out[..., at:at + group] = least.double() + code.double() * width.double()
    return out


def exact(case, seed):
    op = case["op"]
    if op == "attend4":  # the keys and values themselves, not what is stored of them
        return _exact_attention(case, seed)
    s = prepare(case, seed)
    if op == "append4":
        live = (s["slots"] >= 0)[:, None, None]
        q = torch.where(live, _turned(s["q"], s["positions"], case), torch.zeros((), dtype=torch.float64, device="cuda"))
        return tuple(_kept(x, case["group"]) * live for x in (_turned(s["k"], s["positions"], case), s["v"])) + (q,)
    if op == "adapters":
        out, x = s["base"].double(), s["x"].double()
        for i in range(case["adapters"]):
            rows = (s["index"] == i).nonzero()[:, 0]
            out[rows] += (x[rows] @ s["a"][i].double().T @ s["b"][i].double().T) * float(s["scales"][i])
        return out
    x, f = s["x"].double(), case["inner"]
    y = torch.zeros_like(x)
    logits = torch.einsum("nd,ed->ne", x, s["router"].double())
    prob = torch.softmax(logits, -1)
    chosen = torch.zeros(case["tokens"], case["top"], dtype=torch.int32, device="cuda")
    part = torch.zeros(case["tokens"], case["top"], dtype=torch.float64, device="cuda")
    for n, row in enumerate(logits.tolist()):
        mine = sorted(range(len(row)), key=lambda e: (-row[e], e))[:case["top"]]
        chosen[n] = torch.tensor(mine)
        w = prob[n, mine]
        part[n] = w / w.sum() if case["renormalize"] else w
        for e, p in zip(mine, part[n]):
            h = s["gate_up"][e].double() @ x[n]
            act = torch.nn.functional.silu(h[:f]) if case["activation"] == "silu" else torch.nn.functional.gelu(h[:f], approximate="tanh")
            y[n] += p * (s["down"][e].double() @ (act * h[f:]))
    return y, chosen, part


def _exact_attention(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, hk, d, page = TYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    lens = lengths(case)
    lens = [lens[i] for i in torch.randperm(len(lens), generator=g, device="cuda").tolist()]
    pages = sum(-(-n // page) for n in lens) + 3
    free = torch.randperm(pages, generator=g, device="cuda")
    k, v = (torch.randn(pages * page, hk, d, generator=g, device="cuda", dtype=t) for _ in range(2))
    k += 4 * (torch.rand(hk, d, generator=g, device="cuda") < 0.05).to(t)
    q = torch.randn(case["batch"], case["heads"], d, generator=g, device="cuda", dtype=t).double()
    out = torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for b, n in enumerate(lens):
        own_pages = free[first:first + -(-n // page)]
        first += len(own_pages)
        if not n:
            continue
        j = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        at = own_pages[j // page] * page + j % page
        keys, values = (_kept(x[at], case["group"]).transpose(0, 1) for x in (k, v))  # [kv heads, keys, dim]
        score = q[b].view(hk, case["heads"] // hk, d) @ keys.transpose(1, 2) * d ** -0.5
        lse[b] = torch.logsumexp(score, -1).flatten()
        out[b] = (torch.softmax(score, -1) @ values).flatten(0, 1)
    return (out, lse) if case["lse"] else out
