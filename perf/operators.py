"""The decoder operators beside the quantized linears, as workloads: the fused residual norm, rotary
positions with the append to the paged cache, attention over that cache, and copies of its pages.

Each case is a dict of plain values.  ``prepare`` makes the inputs a serving program has in hand,
``run`` makes one call -- of qlinear where ``own`` is true, else the operator's plain form in
elementary torch operations -- and ``exact`` is the definition in 64 bits."""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-5


_module = None


def _qlinear():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "mlx-gen_b200"))
        import qlinear
        _module = qlinear
    return _module


# ----------------------------------------------------------------------------- cases

def listed():
    llama = dict(op="attention", dtype="bf16", hq=24, hkv=8, d=128, causal=True, window=0)
    return [
        # one token of a short prompt-refine chat (Llama-3.2-3B heads): latency counts
        dict(llama, name="attention_token", batch=1, q_min=1, q_max=1, ctx_min=776, ctx_max=776, page=16),
        # a serving batch in decode, every sequence at its own length
        dict(llama, name="attention_decode", batch=64, q_min=1, q_max=1, ctx_min=311, ctx_max=8003, page=16),
        # two long documents in decode: few rows over a long axis
        dict(llama, name="attention_long", batch=2, q_min=1, q_max=1, ctx_min=130001, ctx_max=131070, page=64),
        # a chunk of a long prompt over what is already cached
        dict(llama, name="attention_chunk", batch=1, q_min=512, q_max=512, ctx_min=16021, ctx_max=16021, page=32),
        # a whole prompt at once
        dict(llama, name="attention_prompt", batch=1, q_min=4096, q_max=4096, ctx_min=0, ctx_max=0, page=64),
        # continuous batching: single tokens beside chunks of other prompts, small heads, a sliding window, f16
        dict(op="attention", name="attention_mixed", dtype="f16", batch=17, q_min=1, q_max=389, ctx_min=0, ctx_max=3100,
             hq=32, hkv=8, d=64, causal=True, window=1024, page=16),
        # the residual stream of one decode step of 4 sequences (Llama-3.2-3B width)
        dict(op="norm", name="norm_token", rows=4, d=3072, dtype="bf16", residual="bf16", post=False, gate=False, scale=False),
        # Z-Image's block: norm of the branch, gate, residual, norm before the next branch, 4096 + 512 tokens
        dict(op="norm", name="norm_image", rows=4608, d=3840, dtype="bf16", residual="bf16", post=True, gate=True, scale=True),
        # one decode step of 4 sequences: the step's q, k, v from the fused projection
        dict(op="rope", name="rope_token", tokens=4, hq=24, hkv=8, d=128, rot=128, layout="half", cache=True, page=16, dtype="bf16"),
        # a whole prompt appended to the cache
        dict(op="rope", name="rope_prompt", tokens=4096, hq=24, hkv=8, d=128, rot=128, layout="half", cache=True, page=16, dtype="bf16"),
        # forking three sequences: each copies its last, partly filled page, in all 28 layers
        dict(op="pages", name="pages_fork", copies=3, total=96, layers=28, hkv=8, d=128, page=16, dtype="bf16"),
        # compacting a pool after most sequences have left
        dict(op="pages", name="pages_compact", copies=213, total=512, layers=28, hkv=8, d=128, page=16, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "norm", "rope", "pages"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        d = rng.choice([rng.randrange(64, 8193, 8), 8 * _log(rng, 8, 1024), _log(rng, 33, 5001)])
        post = rng.random() < 0.5
        return dict(op=op, rows=_log(rng, 1, 17_000_000 // d), d=d, dtype=dtype, residual=rng.choice([dtype, "f32"]),
                    post=post, gate=post and rng.random() < 0.6, scale=rng.random() < 0.4)
    hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        d = rng.choice([64, 96, 128, 256])
        tokens = _log(rng, 1, min(6000, 20_000_000 // (d * hkv * (group + 2))))
        return dict(op=op, tokens=tokens, hq=hkv * group, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2]),
                    layout=rng.choice(["half", "interleaved"]), cache=rng.random() < 0.7, page=page, dtype=dtype)
    if op == "pages":
        d, layers = rng.choice([64, 128]), _log(rng, 1, 40)
        hkv = rng.choice([2, 4, 8])
        most = 390_000_000 // (layers * 2 * hkv * page * d * 2)
        copies = _log(rng, 1, max(1, min(600, most)))
        return dict(op=op, copies=copies, total=copies * 2 + rng.randrange(1, 60), layers=layers, hkv=hkv, d=d, page=page, dtype=dtype)
    mode = rng.choice(["token", "decode", "chunk", "prompt", "mixed"])
    while True:
        c = dict(op=op, dtype=dtype, hq=hkv * group, hkv=hkv, d=rng.choice([64, 128, 128]), causal=True,
                 window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), page=page)
        batch = 1 if mode == "token" else _log(rng, 1, 128) if mode == "decode" else _log(rng, 1, 24)
        top = _log(rng, 1, 130000)
        q = 1 if mode in ("token", "decode") else _log(rng, 2, 4096)
        c.update(batch=batch, q_max=q, q_min=q if mode != "mixed" else 1)
        c.update(ctx_max=0 if mode == "prompt" else top, ctx_min=0 if mode == "prompt" else rng.randrange(0, top + 1))
        if mode in ("chunk", "prompt"):
            c["causal"] = rng.random() < 0.8
        if not c["causal"]:
            c["window"] = 0
        w, rows = work(c), batch * c["hq"] * q * (c["ctx_max"] + q)
        if w["bytes"] <= 1.0e9 and w["flops"] <= 1.0e11 and rows <= 4e8 and batch * (c["ctx_max"] + q) * hkv * c["d"] <= 5e8:
            return c


def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, both among them, in an order that mixes short and long."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    while math.gcd(step, n) > 1:
        step += 1
    return [v[(i * step) % n] for i in range(n)]


def _lens(c):
    q = _spread(c["q_min"], c["q_max"], c["batch"], 5)
    ctx = _spread(c["ctx_min"], c["ctx_max"], c["batch"], 7)
    return q, [a + b for a, b in zip(q, ctx)]


# ----------------------------------------------------------------------------- work

def _visible(c, q, kv):
    """Pairs of a new token and a cached position that it sees."""
    if not c["causal"]:
        return q * kv
    if not c["window"]:
        return q * (kv - q) + q * (q + 1) // 2
    return sum(min(c["window"], kv - q + i + 1) for i in range(q))


def _read(c, q, kv):
    """Cached positions that at least one of the q new tokens sees."""
    return kv if not c["window"] else min(kv, c["window"] + q - 1)


def work(c):
    e = _SIZE[c["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["d"]
        rows = c["d"] * e * (1 + c["post"] + c["gate"] + c["scale"])
        return {"bytes": n * 2 * (e + _SIZE[c["residual"]]) + rows, "flops": n * (5 + 4 * c["post"] + c["gate"] + c["scale"])}
    if c["op"] == "rope":
        heads = c["hq"] + c["hkv"] * (2 if c["cache"] else 1)
        return {"bytes": c["tokens"] * (heads * c["d"] * e * 2 + c["rot"] * 4 + 8 + 8 * c["cache"]),
                "flops": c["tokens"] * (c["hq"] + c["hkv"]) * c["rot"] * 3}
    if c["op"] == "pages":
        return {"bytes": 2 * c["copies"] * c["layers"] * 2 * c["hkv"] * c["page"] * c["d"] * e, "flops": 0}
    q, kv = _lens(c)
    pairs = sum(_visible(c, a, b) for a, b in zip(q, kv))
    read = sum(_read(c, a, b) for a, b in zip(q, kv))
    return {"bytes": 2 * sum(q) * c["hq"] * c["d"] * e + 2 * read * c["hkv"] * c["d"] * e, "flops": 4 * pairs * c["hq"] * c["d"]}


# ----------------------------------------------------------------------------- inputs

def _randn(g, shape, dtype, std=1.0):
    """Normal values in the given type, made in pieces (no full-size f32 copy)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        part = flat[i:i + (1 << 26)]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
    return out


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]
    s = {"case": c}
    if c["op"] == "norm":
        m, d = c["rows"], c["d"]
        s["y"] = _randn(g, (m, d), dt, 0.5)
        s["residual"] = _randn(g, (m, d), _DT[c["residual"]], 2.0)
        s["weight"] = 1 + _randn(g, (d,), dt, 0.2)
        s["post"] = 1 + _randn(g, (d,), dt, 0.2) if c["post"] else None
        s["gate"] = torch.tanh(_randn(g, (1, d), dt, 0.7)) if c["gate"] else None
        s["scale"] = _randn(g, (1, d), dt, 0.3) if c["scale"] else None
        s["alpha"] = 0.7071
        return s
    if c["op"] == "rope":
        t, hq, hkv, d, page = c["tokens"], c["hq"], c["hkv"], c["d"], c["page"]
        # q, k and v are views of the fused projection's rows
        qkv = _randn(g, (t, (hq + 2 * hkv) * d), dt)
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
        # rows of cosines and sines, base 500000, for 8192 positions
        f = 500000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
        a = torch.arange(8192, dtype=torch.float64, device="cuda")[:, None] * f
        s["table"] = torch.cat([a.cos(), a.sin()], 1).float()
        first = int(torch.randint(0, 8192 - t + 1, (1,), generator=g, device="cuda")) if t <= 8192 else 0
        s["positions"] = torch.arange(first, first + t, device="cuda")
        if c["cache"]:
            pages = -(-t // page) + 3
            s["k_cache"] = _randn(g, (pages, hkv, page, d), dt)
            s["v_cache"] = _randn(g, (pages, hkv, page, d), dt)
            order = torch.randperm(pages, generator=g, device="cuda")
            i = torch.arange(t, device="cuda") + min(5, 3 * page - 1)
            s["slots"] = order[i // page] * page + i % page
        return s
    if c["op"] == "pages":
        s["pool"] = _randn(g, (c["layers"], 2, c["total"], c["hkv"], c["page"], c["d"]), dt)
        order = torch.randperm(c["total"], generator=g, device="cuda")
        s["src"], s["dst"] = order[:c["copies"]].clone(), order[c["copies"]:2 * c["copies"]].clone()
        # the program's own lists (its page tables live on the host)
        s["src_list"], s["dst_list"] = s["src"].tolist(), s["dst"].tolist()
        return s
    q, kv = _lens(c)
    per = [-(-n // c["page"]) for n in kv]
    total = sum(per) + 1
    s["q"] = _randn(g, (sum(q), c["hq"], c["d"]), dt)
    s["k_cache"] = _randn(g, (total, c["hkv"], c["page"], c["d"]), dt)
    s["v_cache"] = _randn(g, (total, c["hkv"], c["page"], c["d"]), dt)
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    table = torch.full((c["batch"], max(per)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s["page_table"] = table.cuda()
    starts = torch.zeros(c["batch"] + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q).cumsum(0)
    s["q_starts"] = starts.cuda()
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32).cuda()
    s["max_q"], s["max_kv"] = max(q), max(kv)
    return s


# ----------------------------------------------------------------------------- one pass

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _norm_own(s):
    h, r = _qlinear().norm_residual(s["y"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"],
                                    scale=s["scale"], alpha=s["alpha"], eps=_EPS)
    return {"h": h, "r": r}


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)


def _norm_plain(s):
    u = s["y"].float()
    if s["post"] is not None:
        u = _rms(u) * s["post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    r = s["residual"].float() + s["alpha"] * u
    h = _rms(r) * s["weight"].float()
    if s["scale"] is not None:
        h = h * (1 + s["scale"].float())
    return {"h": h.to(s["y"].dtype), "r": r.to(s["residual"].dtype)}


def _rope_own(s):
    c, ql = s["case"], _qlinear()
    if not c["cache"]:
        q, k = ql.rope(s["q"], s["k"], s["table"], s["positions"], layout=c["layout"])
        return {"q": q, "k": k}
    q = ql.rope_append(s["q"], s["k"], s["v"], s["table"], s["positions"], s["k_cache"], s["v_cache"], s["slots"],
                       layout=c["layout"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rotate_plain(x, cos, sin, layout):
    n = cos.shape[-1]
    y = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = y[..., :n], y[..., n:2 * n]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([rot, y[..., 2 * n:]], -1).to(x.dtype)


def _rope_plain(s):
    c = s["case"]
    row = s["table"][s["positions"]]
    cos, sin = row.chunk(2, -1)
    q, k = _rotate_plain(s["q"], cos, sin, c["layout"]), _rotate_plain(s["k"], cos, sin, c["layout"])
    if not c["cache"]:
        return {"q": q, "k": k}
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_cache"][page, :, at] = k
    s["v_cache"][page, :, at] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _pages_own(s):
    _qlinear().copy_pages(s["pool"], s["src_list"], s["dst_list"])
    return {"pool": s["pool"]}


def _pages_plain(s):
    s["pool"][:, :, s["dst"]] = s["pool"][:, :, s["src"]]
    return {"pool": s["pool"]}


def _attention_own(s):
    c = s["case"]
    o = _qlinear().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["q_starts"], s["kv_lens"],
                                   max_q=s["max_q"], max_kv=s["max_kv"], causal=c["causal"], window=c["window"])
    return {"o": o}


def _attention_plain(s):
    """All sequences padded to the longest, the whole score matrix, one softmax."""
    c = s["case"]
    b, page, hkv, d = c["batch"], c["page"], c["hkv"], c["d"]
    g, n, m = c["hq"] // hkv, s["max_kv"], s["max_q"]
    q_lens = s["q_starts"][1:] - s["q_starts"][:-1]
    i, j = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    table = s["page_table"].long().clamp(min=0)
    k = s["k_cache"][table].transpose(1, 2).reshape(b, hkv, -1, d)[:, :, :n].float()
    v = s["v_cache"][table].transpose(1, 2).reshape(b, hkv, -1, d)[:, :, :n].float()
    rows = (s["q_starts"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(b, m, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * m, d)
    x = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hkv, g, m, n)
    at = (s["kv_lens"] - q_lens)[:, None] + i
    seen = j[None, None] < s["kv_lens"][:, None, None]
    if c["causal"]:
        seen = seen & (j <= at[..., None])
        if c["window"]:
            seen = seen & (j > at[..., None] - c["window"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(b, hkv, g * m, n) @ v).view(b, hkv, g, m, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, m, c["hq"], d)
    return {"o": o[i < q_lens[:, None]].to(s["q"].dtype)}


_own = {"norm": _norm_own, "rope": _rope_own, "pages": _pages_own, "attention": _attention_own}
_plain = {"norm": _norm_plain, "rope": _rope_plain, "pages": _pages_plain, "attention": _attention_plain}


# ----------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    if c["op"] == "norm":
        n = c["d"]
        y, r = s["y"].double(), s["residual"].double()
        if s["post"] is not None:
            y = torch.einsum("md,d,m->md", y, s["post"].double(), (torch.einsum("md,md->m", y, y) / n + _EPS) ** -0.5)
        if s["gate"] is not None:
            y = torch.einsum("md,d->md", y, s["gate"].double()[0])
        r = torch.add(r, y, alpha=s["alpha"])
        w = s["weight"].double() if s["scale"] is None else s["weight"].double() * (1 + s["scale"].double()[0])
        return {"h": torch.einsum("md,d,m->md", r, w, (torch.einsum("md,md->m", r, r) / n + _EPS) ** -0.5), "r": r}
    if c["op"] == "rope":
        half = c["rot"] // 2
        z = torch.complex(s["table"][:, :half].double(), s["table"][:, half:].double())[s["positions"]][:, None]

        def turn(x):
            x = x.double().clone()
            p = x[..., :c["rot"]]
            p = p.unflatten(-1, (2, half)).transpose(-1, -2) if c["layout"] == "half" else p.unflatten(-1, (half, 2))
            p = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
            x[..., :c["rot"]] = (p.transpose(-1, -2) if c["layout"] == "half" else p).flatten(-2)
            return x

        q, k = turn(s["q"]), turn(s["k"])
        if not c["cache"]:
            return {"q": q, "k": k}
        kc, vc = (s[x].double().transpose(1, 2).reshape(-1, c["hkv"], c["d"]) for x in ("k_cache", "v_cache"))
        kc[s["slots"]], vc[s["slots"]] = k, s["v"].double()
        back = [x.view(-1, c["page"], c["hkv"], c["d"]).transpose(1, 2) for x in (kc, vc)]
        return {"q": q, "k_cache": back[0], "v_cache": back[1]}
    if c["op"] == "pages":
        pool = s["pool"]
        for a, b in zip(s["src_list"], s["dst_list"]):
            pool[:, :, b].copy_(pool[:, :, a])
        return {"pool": pool}
    q, kv = _lens(c)
    out = torch.zeros(sum(q), c["hq"], c["d"], dtype=torch.float64, device="cuda")
    g, at = c["hq"] // c["hkv"], 0
    for b in range(c["batch"]):
        pages = s["page_table"][b, :-(-kv[b] // c["page"])].long()
        j = torch.arange(kv[b], device="cuda")[None, :]
        i = kv[b] - q[b] + torch.arange(q[b], device="cuda")[:, None]
        hide = torch.zeros(q[b], kv[b], dtype=torch.bool, device="cuda")
        if c["causal"]:
            hide |= j > i
            if c["window"]:
                hide |= i - j >= c["window"]
        for h in range(c["hkv"]):
            k = s["k_cache"][pages, h].reshape(-1, c["d"])[:kv[b]].double()
            v = s["v_cache"][pages, h].reshape(-1, c["d"])[:kv[b]].double()
            for e in range(h * g, h * g + g):
                x = s["q"][at:at + q[b], e].double() @ k.T / c["d"] ** 0.5
                out[at:at + q[b], e] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
        at += q[b]
    return {"o": out}
