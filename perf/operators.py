"""The attention operators of tccl_amd as timed and compared cases: what each stands for, its plain form, its value in 64 bits and its work.

Five kinds of case, a user's steps when the ranks of a group hold parts of a sequence:

``norm_rope``   the ranks' partial query/key/value projections are summed, queries and keys normed per head and rotated
``norm_grad``   the same operator's backward pass: gradients of the projection and of the two norm weights
``cache``       new tokens are written into a paged cache that spans the ranks, and whole sequences are read back from it
``attention``   one new token per sequence attends to the paged cache of all ranks
``join``        the ranks' partial attentions over their own parts become the whole one (a softmax-weighted all-reduce)
"""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f32": 4, "e4m3": 1}
EPS = 1e-6
LEAST_EXPONENT = -110


def listed():
    return [
        # a decode step of 32 sequences: eight ranks' partial projections; latency counts
        dict(name="norm_rope decode w8", kind="norm_rope", world=8, tokens=32, q_heads=32, k_heads=8, v_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bf16", far=32768),
        # a prompt chunk of an odd length over eight ranks
        dict(name="norm_rope prompt w8", kind="norm_rope", world=8, tokens=4099, q_heads=32, k_heads=8, v_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bf16", far=131072),
        # float32 training forward of one rank: a quarter of each head is rotated, neighbouring pairs, no values behind the keys
        dict(name="norm_rope f32 interleaved", kind="norm_rope", world=1, tokens=8191, q_heads=16, k_heads=4, v_heads=0, dim=256, rotary=64,
             interleaved=True, dtype="f32", far=8191),
        # the training step's backward pass on one rank
        dict(name="norm_grad training", kind="norm_grad", world=1, tokens=8192, q_heads=32, k_heads=8, v_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bf16", far=8192),
        # a small float32 backward pass over four partial projections
        dict(name="norm_grad f32 w4", kind="norm_grad", world=4, tokens=777, q_heads=12, k_heads=12, v_heads=12, dim=64, rotary=32,
             interleaved=True, dtype="f32", far=4096),
        # chunked prefill: 1,024 new tokens each behind histories of up to 8,192, kept in 8 bits, then read back whole
        dict(name="cache chunk e4m3", kind="cache", world=8, batch=8, history=8192, new=1024, heads=8, dim=128, page=64, store="e4m3",
             dtype="bf16"),
        # a decode step's write of one token each, and the short sequences read back for a migration
        dict(name="cache decode bf16", kind="cache", world=4, batch=128, history=400, new=1, heads=4, dim=64, page=16, store="bf16",
             dtype="bf16"),
        # one user's chat: latency
        dict(name="attention single", kind="attention", world=2, batch=1, longest=1500, q_heads=32, k_heads=8, dim=128, page=16,
             store="bf16"),
        # a serving batch of ragged lengths (one is empty) over an 8-bit cache on eight ranks
        dict(name="attention batch e4m3", kind="attention", world=8, batch=64, longest=8192, q_heads=64, k_heads=8, dim=128, page=64,
             store="e4m3"),
        # three very long documents, all query heads on one key head
        dict(name="attention long shared", kind="attention", world=8, batch=3, longest=200003, q_heads=24, k_heads=1, dim=256, page=128,
             store="bf16"),
        # the join after a decode step
        dict(name="join decode w8", kind="join", world=8, rows=2048, dim=128, dtype="bf16"),
        # the join of a whole float32 prompt's heads over four ranks
        dict(name="join prompt f32 w4", kind="join", world=4, rows=131071, dim=64, dtype="f32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "norm_grad", "cache", "attention", "join"])
    dim = rng.choice([64, 128, 256])
    world = rng.randint(1, 8)
    if kind in ("norm_rope", "norm_grad"):
        k_heads = rng.choice([1, 2, 3, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 4, 5])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        row = world * (q_heads + 2 * k_heads) * dim * WIDTH[dtype]
        return dict(kind=kind, world=world, tokens=_spread(rng, 1, min(8192, max(2, 300_000_000 // row))), q_heads=q_heads, k_heads=k_heads,
                    v_heads=rng.choice([0, k_heads]), dim=dim, rotary=rng.choice([dim, dim // 2, 32]), interleaved=rng.random() < 0.5,
                    dtype=dtype, far=_spread(rng, 100, 1_000_000))
    if kind == "cache":
        heads = rng.choice([1, 2, 4, 8])
        batch = _spread(rng, 1, 64)
        most = max(2, min(8192, 60_000 * 1024 // (heads * dim * batch)))
        return dict(kind=kind, world=world, batch=batch, history=_spread(rng, 1, most), new=_spread(rng, 1, max(2, min(1024, most // 4))),
                    heads=heads, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), store=rng.choice(["bf16", "e4m3"]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "attention":
        k_heads = rng.choice([1, 2, 4, 8])
        batch = _spread(rng, 1, 128)
        most = max(17, min(200_000, 500_000 * 1024 // (k_heads * dim * batch)))
        return dict(kind=kind, world=world, batch=batch, longest=_spread(rng, 16, most), q_heads=k_heads * rng.choice([1, 2, 4, 7, 8, 16]),
                    k_heads=k_heads, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), store=rng.choice(["bf16", "e4m3"]))
    dtype = rng.choice(["bf16", "f32"])
    return dict(kind=kind, world=world, rows=_spread(rng, 1, 33_000_000 // (dim * WIDTH[dtype] * world)), dim=dim, dtype=dtype)


# ---------------------------------------------------------------- inputs

def _length_values(batch, longest):
    """Ragged: evenly from a quarter of the longest to the longest; of eight or more sequences one is empty."""
    empty = int(batch >= 8)
    full = batch - empty
    least = max(1, longest // 4)
    return [0] * empty + [longest - (longest - least) * i // max(1, full - 1) for i in range(full)]


def _lengths(rng, batch, longest):
    n = torch.tensor(_length_values(batch, longest), device=DEV)
    return n[torch.randperm(batch, generator=rng, device=DEV)]


def _table(rng, world, batch, longest, page):
    """A page table over pages in random order on all ranks, and the pages that each rank has."""
    width = -(-longest // page)
    each = -(-batch * width // world)
    ids = torch.randperm(world * each, generator=rng, device=DEV)[: batch * width]
    return ids.view(batch, width).to(torch.int32), each


def _slots(table, page, start, stop):
    """Slots (page * page size + place in the page) of tokens [start[b], stop[b]) of every sequence, one sequence behind the other."""
    width = table.shape[1] * page
    at = torch.arange(width, device=DEV).expand(table.shape[0], width)
    slot = table.long().repeat_interleave(page, 1) * page + at % page
    return slot[(at >= start[:, None]) & (at < stop[:, None])].contiguous()


def prepare(case, seed):
    rng = torch.Generator(device=DEV)
    rng.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=rng, device=DEV, dtype=torch.float32).to(dtype)

    c = dict(case)
    kind = c["kind"]
    s = {"case": c}
    if kind in ("norm_rope", "norm_grad"):
        dtype = DTYPES[c["dtype"]]
        heads = c["q_heads"] + c["k_heads"] + c["v_heads"]
        s["parts"] = [normal(c["tokens"], heads * c["dim"], dtype=dtype) for _ in range(c["world"])]
        s["q_weight"] = (1 + 0.2 * normal(c["dim"])).to(dtype)
        s["k_weight"] = (1 + 0.2 * normal(c["dim"])).to(dtype)
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=rng, device=DEV)
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, c["rotary"], 2, device=DEV, dtype=torch.float64) / c["rotary"])
        if kind == "norm_grad":
            s["grads"] = [normal(c["tokens"], n, c["dim"], dtype=dtype) for n in (c["q_heads"], c["k_heads"], c["v_heads"])]
        if own:
            import tccl_amd
            s["group"] = tccl_amd.register(s["parts"])
    elif kind == "cache":
        history = _lengths(rng, c["batch"], c["history"])
        table, each = _table(rng, c["world"], c["batch"], c["history"] + c["new"], c["page"])
        old = _slots(table, c["page"], torch.zeros_like(history), history)
        s["new_slots"] = _slots(table, c["page"], history, history + c["new"])
        s["all_slots"] = _slots(table, c["page"], torch.zeros_like(history), history + c["new"])
        dtype = DTYPES[c["dtype"]]
        _store(s, each, old, normal(len(old), c["heads"], c["dim"], dtype=dtype), normal(len(old), c["heads"], c["dim"], dtype=dtype))
        s["k"] = normal(len(s["new_slots"]), c["heads"], c["dim"], dtype=dtype) * 3
        s["v"] = normal(len(s["new_slots"]), c["heads"], c["dim"], dtype=dtype)
    elif kind == "attention":
        lengths = _lengths(rng, c["batch"], c["longest"])
        s["table"], each = _table(rng, c["world"], c["batch"], c["longest"], c["page"])
        s["lengths"] = lengths.to(torch.int32)
        s["longest"] = c["longest"]
        slots = _slots(s["table"], c["page"], torch.zeros_like(lengths), lengths)
        c["heads"] = c["k_heads"]
        _store(s, each, slots, normal(len(slots), c["k_heads"], c["dim"], dtype=torch.bfloat16),
               normal(len(slots), c["k_heads"], c["dim"], dtype=torch.bfloat16))
        s["q"] = normal(c["batch"], c["q_heads"], c["dim"], dtype=torch.bfloat16)
    else:
        dtype = DTYPES[c["dtype"]]
        s["outs"] = [normal(c["rows"], c["dim"], dtype=dtype) for _ in range(c["world"])]
        s["lses"] = [3 * normal(c["rows"]) for _ in range(c["world"])]
        for r in range(c["world"]):     # a rank that holds no token of a sequence: here every eleventh row, shifted by rank
            s["lses"][r][r::11] = -math.inf
        if own:
            import tccl_amd
            s["groups"] = tccl_amd.register(s["outs"]), tccl_amd.register(s["lses"])
    return s


def _store(s, each, slots, k, v):
    """The cache with what earlier calls wrote into it: the framework's own, or plain rows by slot (8-bit codes beside their exponents)."""
    c = s["case"]
    if own:
        import tccl_amd
        s["cache"] = tccl_amd.PagedCache(c["world"], each, c["page"], c["heads"], c["dim"],
                                         dtype=torch.bfloat16 if c["store"] == "bf16" else torch.float8_e4m3fn, device=DEV)
        tccl_amd.cache_write(s["cache"], k, v, slots)
        return
    shape = (c["world"] * each * c["page"], c["heads"], c["dim"])
    for name, x in (("k", k), ("v", v)):
        if c["store"] == "bf16":
            s[name + "_rows"] = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        else:
            s[name + "_rows"] = torch.zeros(shape, dtype=torch.uint8, device=DEV)
            s[name + "_exponents"] = torch.zeros(shape[:2] + (1,), dtype=torch.int32, device=DEV)
        _put(s, name, slots, x)


# ---------------------------------------------------------------- the plain forms

def _put(s, name, slots, x):
    if s["case"]["store"] == "bf16":
        s[name + "_rows"][slots] = x.to(torch.bfloat16)
        return
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))          # the largest is m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.clamp(e - 9 + (m > 0.875).int(), min=LEAST_EXPONENT)
    s[name + "_rows"][slots] = torch.ldexp(x, -e).to(torch.float8_e4m3fn).view(torch.uint8)
    s[name + "_exponents"][slots] = e.int()


def _get(s, name, slots):
    rows = s[name + "_rows"][slots]
    if s["case"]["store"] == "bf16":
        return rows.float()
    return torch.ldexp(rows.view(torch.float8_e4m3fn).float(), s[name + "_exponents"][slots])


def _angles(s):
    a = s["positions"].double()[:, None] * s["inv_freq"]
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _pairs(x, rotary, interleaved):
    x = x[..., :rotary]
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., : rotary // 2], x[..., rotary // 2:])


def _rotated(x, cos, sin, rotary, interleaved):
    a, b = _pairs(x, rotary, interleaved)
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1 if interleaved else -2).flatten(-2)
    return torch.cat((y, x[..., rotary:]), -1)


def _heads(s):
    c = s["case"]
    x = torch.stack(s["parts"]).float().sum(0).view(c["tokens"], -1, c["dim"])
    return x.split((c["q_heads"], c["k_heads"], c["v_heads"]), 1)


def _norm_rope(s):
    c = s["case"]
    dtype = DTYPES[c["dtype"]]
    q, k, v = _heads(s)
    cos, sin = _angles(s)

    def one(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        return _rotated(y, cos, sin, c["rotary"], c["interleaved"]).to(dtype)

    return one(q, s["q_weight"]), one(k, s["k_weight"]), v.to(dtype)


def _norm_grad(s):
    c = s["case"]
    q, k, _ = _heads(s)
    cos, sin = _angles(s)

    def one(x, w, dy):
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        g = _rotated(dy.float(), cos, -sin, c["rotary"], c["interleaved"])
        u = g * w.float()
        return r * (u - n * (u * n).mean(-1, keepdim=True)), (g * n).sum((0, 1), dtype=torch.float64).float()

    dq, dqw = one(q, s["q_weight"], s["grads"][0])
    dk, dkw = one(k, s["k_weight"], s["grads"][1])
    dx = torch.cat((dq, dk, s["grads"][2].float()), 1).flatten(1)
    return dx.to(DTYPES[c["dtype"]]), dqw, dkw


def _attention(s):
    c = s["case"]
    group = c["q_heads"] // c["k_heads"]
    at = torch.arange(s["longest"], device=DEV)
    valid = at < s["lengths"][:, None]
    slots = s["table"].long()[:, at // c["page"]] * c["page"] + at % c["page"]
    slots = torch.where(valid, slots, 0)
    q = s["q"].float().view(c["batch"], c["k_heads"], group, c["dim"])
    k = _get(s, "k", slots).permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(q, k) / math.sqrt(c["dim"])
    del k
    score = score.masked_fill(~valid[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = torch.where(valid[:, :, None, None], _get(s, "v", slots), 0.0).transpose(1, 2).contiguous()
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out.flatten(1, 2).to(torch.bfloat16), (top + torch.log(total)).flatten(1)


def _join(s):
    lse = torch.stack(s["lses"])
    top = lse.amax(0)
    top = torch.where(torch.isfinite(top), top, 0.0)
    w = torch.exp(lse - top)
    total = w.sum(0)
    out = (torch.stack(s["outs"]).float() * w[..., None]).sum(0) / torch.where(total > 0, total, 1.0)[:, None]
    return out.to(DTYPES[s["case"]["dtype"]]), top + torch.log(total)


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        import tccl_amd
        if kind == "norm_rope":
            return tccl_amd.qk_norm_rope(s["parts"][0], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], c["q_heads"], c["k_heads"],
                                         eps=EPS, interleaved=c["interleaved"])
        if kind == "norm_grad":
            return tccl_amd.qk_norm_rope_backward(*s["grads"], s["parts"][0], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"],
                                                  eps=EPS, interleaved=c["interleaved"])
        if kind == "cache":
            tccl_amd.cache_write(s["cache"], s["k"], s["v"], s["new_slots"])
            return tccl_amd.cache_read(s["cache"], s["all_slots"], dtype=DTYPES[c["dtype"]])
        if kind == "attention":
            return tccl_amd.decode_attention(s["q"], s["cache"], s["table"], s["lengths"], max_length=s["longest"], return_lse=True)
        return tccl_amd.attention_all_reduce(s["outs"][0], s["lses"][0])
    if kind == "norm_rope":
        return _norm_rope(s)
    if kind == "norm_grad":
        return _norm_grad(s)
    if kind == "cache":
        _put(s, "k", s["new_slots"], s["k"])
        _put(s, "v", s["new_slots"], s["v"])
        return _get(s, "k", s["all_slots"]).to(s["k"].dtype), _get(s, "v", s["all_slots"]).to(s["v"].dtype)
    if kind == "attention":
        return _attention(s)
    return _join(s)


# ---------------------------------------------------------------- work

def work(case):
    c, kind = case, case["kind"]
    if kind in ("norm_rope", "norm_grad"):
        heads = c["q_heads"] + c["k_heads"] + c["v_heads"]
        row = heads * c["dim"] * WIDTH[c["dtype"]]
        moved = (c["world"] + 1) * row if kind == "norm_rope" else 2 * row + (c["world"] * (heads - c["v_heads"]) * row) // heads
        small = 2 * c["dim"] * WIDTH[c["dtype"]] + (8 * c["dim"] if kind == "norm_grad" else 0) + 4 * c["rotary"]
        each = c["world"] + (8 if kind == "norm_rope" else 18)
        return {"bytes": c["tokens"] * (moved + 8) + small, "flops": c["tokens"] * heads * c["dim"] * each}
    if kind == "join":
        row = c["dim"] * WIDTH[c["dtype"]] + 4
        return {"bytes": (c["world"] + 1) * c["rows"] * row, "flops": 2 * c["world"] * c["rows"] * c["dim"]}
    tokens = sum(_length_values(c["batch"], c["history"] if kind == "cache" else c["longest"]))
    kept = c["dim"] * WIDTH[c["store"]] + (c["store"] == "e4m3")
    if kind == "cache":
        new = c["batch"] * c["new"]
        plain = c["dim"] * WIDTH[c["dtype"]]
        moved = 2 * c["heads"] * (new * (plain + kept) + (tokens + new) * (plain + kept))
        return {"bytes": moved + 8 * (tokens + 2 * new), "flops": 2 * c["heads"] * c["dim"] * (tokens + 3 * new)}
    small = c["batch"] * (c["q_heads"] * (4 * c["dim"] + 4) + 4) + 4 * tokens // c["page"]
    return {"bytes": 2 * tokens * c["k_heads"] * kept + small, "flops": 4 * tokens * c["q_heads"] * c["dim"]}


# ---------------------------------------------------------------- the operators' values in 64 bits

def _turned(x, angle, rotary, interleaved):
    """The rotation as a product of complex numbers."""
    head = x[..., :rotary]
    z = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = torch.view_as_real(z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., rotary:]), -1)


def _nearest_e4m3(x):
    """What 8 bits with one exponent per row hold of x: the nearest multiple of the step at each value's magnitude, ties to the even one."""
    largest = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(largest / 448))
    e = torch.where(448 * torch.exp2(e - 1) >= largest, e - 1, torch.where(448 * torch.exp2(e) < largest, e + 1, e))
    scale = torch.exp2(torch.clamp(e, min=float(LEAST_EXPONENT)))
    y = x / scale
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0**-20))), min=-6.0) - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    c, kind = s["case"], case["kind"]
    if kind in ("norm_rope", "norm_grad"):
        x = sum(p.double() for p in s["parts"])
        weights = [s["q_weight"].double(), s["k_weight"].double()]
        angle = torch.outer(s["positions"].double(), s["inv_freq"])
        grad = kind == "norm_grad"
        if grad:
            x.requires_grad_()
            weights[0].requires_grad_()
            weights[1].requires_grad_()
        q, k, v = x.view(c["tokens"], -1, c["dim"]).split((c["q_heads"], c["k_heads"], c["v_heads"]), 1)
        y = [_turned(w * h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS), angle, c["rotary"], c["interleaved"])
             for h, w in ((q, weights[0]), (k, weights[1]))]
        if not grad:
            return y[0], y[1], v
        return torch.autograd.grad((*y, v), (x, *weights), [g.double() for g in s["grads"]])
    if kind == "join":
        lse = torch.stack(s["lses"]).double()
        whole = torch.logsumexp(lse, 0)
        share = torch.nan_to_num(torch.exp(lse - whole))
        return sum(share[r][:, None] * s["outs"][r].double() for r in range(c["world"])), whole
    if kind == "cache":
        # an 8-bit history was made by one rounding in prepare(); the new tokens' rounding is computed here from their values
        held = [_get(s, n, s["all_slots"]).double() for n in ("k", "v")]
        order = torch.argsort(s["all_slots"])
        place = order[torch.searchsorted(s["all_slots"][order], s["new_slots"])]
        for h, n in zip(held, ("k", "v")):
            h[place] = s[n].to(torch.bfloat16).double() if c["store"] == "bf16" else _nearest_e4m3(s[n].double())
        return held[0], held[1]
    outs, lses = [], []
    group = c["q_heads"] // c["k_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device=DEV)
        slots = s["table"][b].long()[at // c["page"]] * c["page"] + at % c["page"]
        k, v = _get(s, "k", slots).double(), _get(s, "v", slots).double()
        o, l = [], []
        for h in range(c["k_heads"]):
            score = s["q"][b, h * group:(h + 1) * group].double() @ k[:, h].T / math.sqrt(c["dim"])
            total = torch.logsumexp(score, -1)
            o.append(torch.exp(score - total[:, None]) @ v[:, h])
            l.append(total)
        outs.append(torch.cat(o))
        lses.append(torch.cat(l))
    return torch.stack(outs), torch.stack(lses)
