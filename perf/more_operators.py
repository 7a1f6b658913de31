"""What stands between one step's logits and the next step's attention, as workloads: sampling from
given random numbers, the step's page tables and slots from the sequences' lengths, and attention
over a window with a few first tokens that stay visible (sinks).

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
    heads = dict(op="sinks", dtype="bf16", hq=24, hkv=8, d=128)
    return [
        # one token of one conversation, nucleus sampling over the whole vocabulary: latency counts
        dict(op="sample", name="sample_token", rows=1, vocab=128256, dtype="bf16", temperature=0.8, top_k=0, top_p=0.95,
             min_p=0.0, each=False),
        # four continuations of one prompt, the usual chat settings
        dict(op="sample", name="sample_forks", rows=4, vocab=128256, dtype="bf16", temperature=0.7, top_k=50, top_p=0.9,
             min_p=0.0, each=False),
        # a serving batch in which every request has its own settings, greedy ones among them
        dict(op="sample", name="sample_batch", rows=64, vocab=128256, dtype="bf16", temperature=1.0, top_k=40, top_p=0.9,
             min_p=0.05, each=True),
        # many samples of one prompt at a high temperature: the nucleus holds much of the vocabulary
        dict(op="sample", name="sample_wide", rows=256, vocab=128256, dtype="bf16", temperature=1.5, top_k=0, top_p=0.98,
             min_p=0.0, each=False),
        # logits in f32 (a head kept in full precision), an odd vocabulary, no filter at all
        dict(op="sample", name="sample_plain", rows=96, vocab=151643, dtype="f32", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, each=False),
        # one decode step of a serving batch, some sequences starting a page
        dict(op="plan", name="plan_decode", batch=64, new_min=1, new_max=1, have_min=311, have_max=8003, page=16),
        # continuous batching: prompts beside single tokens and sequences that wait
        dict(op="plan", name="plan_mixed", batch=203, new_min=0, new_max=613, have_min=0, have_max=4001, page=16),
        # one token of an endless conversation: 1024 positions and 4 first tokens of 100000
        dict(heads, name="sinks_token", batch=1, q_min=1, q_max=1, ctx_min=100003, ctx_max=100003, window=1024, sinks=4, page=16),
        # a batch in decode, every sequence at its own length, most of them past the window
        dict(heads, name="sinks_decode", batch=64, q_min=1, q_max=1, ctx_min=1500, ctx_max=60011, window=2048, sinks=4, page=16),
        # a chunk of a long prompt
        dict(heads, name="sinks_chunk", batch=1, q_min=1024, q_max=1024, ctx_min=30011, ctx_max=30011, window=4096, sinks=64, page=32),
        # a whole prompt at once
        dict(heads, name="sinks_prompt", batch=1, q_min=4096, q_max=4096, ctx_min=0, ctx_max=0, window=1024, sinks=4, page=64),
        # single tokens beside chunks of other prompts, small heads, a narrow window, f16
        dict(op="sinks", name="sinks_mixed", dtype="f16", batch=17, q_min=1, q_max=389, ctx_min=0, ctx_max=9100, hq=32, hkv=8,
             d=64, window=256, sinks=16, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "plan", "sinks", "sinks"])
    if op == "sample":
        vocab = rng.choice([128256, _log(rng, 500, 200000), _log(rng, 30000, 260000)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op=op, rows=_log(rng, 1, max(1, 65_000_000 // (vocab * _SIZE[dtype]))), vocab=vocab, dtype=dtype,
                    temperature=round(math.exp(rng.uniform(math.log(0.3), math.log(2.0))), 3),
                    top_k=rng.choice([0, 0, _log(rng, 1, 2000)]), top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.999), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), each=rng.random() < 0.4)
    if op == "plan":
        batch = _log(rng, 1, 2000)
        new = rng.choice([1, _log(rng, 1, min(4096, 60000 // batch + 1))])
        have = _log(rng, 1, 20000)
        return dict(op=op, batch=batch, new_min=new if rng.random() < 0.5 else min(new, rng.randrange(0, 2)), new_max=new,
                    have_min=rng.randrange(0, have + 1), have_max=have, page=rng.choice([16, 32, 64, 128]))
    mode = rng.choice(["token", "decode", "chunk", "prompt", "mixed"])
    while True:
        hkv = rng.choice([1, 2, 4, 8])
        q = 1 if mode in ("token", "decode") else _log(rng, 2, 4096)
        top = _log(rng, 1, 100000)
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv,
                 d=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128]), window=_log(rng, 16, 8192),
                 sinks=_log(rng, 1, 300), batch=1 if mode == "token" else _log(rng, 1, 128) if mode == "decode" else _log(rng, 1, 24))
        c.update(q_max=q, q_min=q if mode != "mixed" else 1, ctx_max=0 if mode == "prompt" else top,
                 ctx_min=0 if mode == "prompt" else rng.randrange(0, top + 1))
        w, n = work(c), _plain_width(c)
        if (w["bytes"] <= 5.3e8 and w["flops"] <= 5.0e10 and c["batch"] * c["hq"] * q * n <= 4e8
                and c["batch"] * n * c["hkv"] * c["d"] <= 4e8):
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
    """New tokens and lengths (with them) of the sequences of an attention case."""
    q = _spread(c["q_min"], c["q_max"], c["batch"], 5)
    ctx = _spread(c["ctx_min"], c["ctx_max"], c["batch"], 7)
    return q, [a + b for a, b in zip(q, ctx)]


def _counts(c):
    """Lengths before the step and new tokens of the sequences of a planning case."""
    return _spread(c["have_min"], c["have_max"], c["batch"], 7), _spread(c["new_min"], c["new_max"], c["batch"], 5)


# ----------------------------------------------------------------------------- work

def _visible(c, q, kv):
    """Pairs of a new token and a cached position that it sees."""
    w, s, ctx = c["window"], c["sinks"], kv - q
    n = 0
    for p in range(ctx, kv):
        lo = max(0, p + 1 - w)
        n += p + 1 - lo + min(s, lo)
    return n


def _read(c, q, kv):
    """Cached positions that at least one of the q new tokens sees."""
    return min(kv, c["sinks"] + c["window"] + q - 1)


def work(c):
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        # a pass over the logits, one exponential each; the settings and numbers of a row, its token
        return {"bytes": n * _SIZE[c["dtype"]] + c["rows"] * (16 + 16 * c["each"]), "flops": 4 * n}
    if c["op"] == "plan":
        have, new = _counts(c)
        ps, b, t = c["page"], c["batch"], sum(new)
        fresh = sum(-(-(h + n) // ps) - -(-h // ps) for h, n in zip(have, new))
        # lengths, counts, the last page; the pages taken, written to the tables; positions, slots, offsets, lengths
        return {"bytes": b * 12 + fresh * 8 + t * 16 + b * 8 + 16, "flops": 4 * t}
    e = _SIZE[c["dtype"]]
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
    s = {"case": c}

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if c["op"] == "sample":
        b, v = c["rows"], c["vocab"]
        x = _randn(g, (b, v), torch.float32, 2.0)
        # a few tokens stand out, as the likely continuations do
        few = min(v, 24)
        at = (rand(b, few) * v).long()
        x.scatter_(1, at, 5.0 + 9.0 * rand(b, few))
        s["logits"] = x.to(_DT[c["dtype"]])
        s["u"] = rand(b)
        for k in ("temperature", "top_k", "top_p", "min_p"):
            s[k] = c[k]
        if c["each"]:
            # every request its own settings: some greedy, some without one filter or the other
            s["temperature"] = torch.where(rand(b) < 0.15, torch.zeros(b, device="cuda"), c["temperature"] * (0.5 + rand(b)))
            s["top_k"] = torch.where(rand(b) < 0.3, torch.zeros(b, device="cuda"), 1 + 2 * c["top_k"] * rand(b)).int()
            s["top_p"] = torch.where(rand(b) < 0.3, torch.ones(b, device="cuda"), c["top_p"] * (0.6 + 0.4 * rand(b)))
            s["min_p"] = torch.where(rand(b) < 0.5, torch.zeros(b, device="cuda"), 2 * c["min_p"] * rand(b))
        return s
    if c["op"] == "plan":
        have, new = _counts(c)
        ps = c["page"]
        held = [-(-h // ps) for h in have]
        fresh = sum(-(-(h + n) // ps) for h, n in zip(have, new)) - sum(held)
        width = max(-(-(h + n) // ps) for h, n in zip(have, new)) + 3
        order = torch.randperm(sum(held) + fresh + 40, generator=g, device="cuda").int()
        table = torch.full((c["batch"], width), -1, dtype=torch.int32, device="cuda")
        col = torch.arange(width, device="cuda")
        table[col < torch.tensor(held, device="cuda")[:, None]] = order[:sum(held)]
        s.update(page_table=table, free_pages=order[sum(held):].clone(), taken=torch.tensor([7], dtype=torch.int32, device="cuda"),
                 lengths=torch.tensor(have, dtype=torch.int32, device="cuda"),
                 new_tokens=torch.tensor(new, dtype=torch.int32, device="cuda"), max_tokens=max(1, sum(new)))
        return s
    q, kv = _lens(c)
    ps, dt = c["page"], _DT[c["dtype"]]
    # the pages between the first tokens and the window have been freed: their entries say -1
    keep = [sorted(set(range(min(-(-n // ps), -(-c["sinks"] // ps)))) | set(range(max(0, n - a + 1 - c["window"]) // ps, -(-n // ps))))
            for a, n in zip(q, kv)]
    total = sum(map(len, keep)) + 1
    s["q"] = _randn(g, (sum(q), c["hq"], c["d"]), dt)
    s["k_cache"] = _randn(g, (total, c["hkv"], ps, c["d"]), dt)
    s["v_cache"] = _randn(g, (total, c["hkv"], ps, c["d"]), dt)
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    table = torch.full((c["batch"], max(-(-n // ps) for n in kv)), -1, dtype=torch.int32)
    at = 0
    for i, pages in enumerate(keep):
        table[i, pages] = torch.tensor(order[at:at + len(pages)], dtype=torch.int32)
        at += len(pages)
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


def _sample_own(s):
    tokens, logprobs = _qlinear().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                         min_p=s["min_p"], logprobs=True)
    return {"tokens": tokens, "logprobs": logprobs}


def _column(x, like):
    """A setting for all rows, or one for each, as a column in 64 bits."""
    return x.double()[:, None] if isinstance(x, torch.Tensor) else torch.full((1, 1), float(x), dtype=torch.float64, device=like.device)


def _sample_plain(s):
    """One stable sort of every row, then prefix sums (in 64 bits: a sum of 128256 weights next to a border)."""
    x = s["logits"].float()
    t, k, p, m = (_column(s[n], x) for n in ("temperature", "top_k", "top_p", "min_p"))
    v, index = torch.sort(x, dim=-1, descending=True, stable=True)
    n, v = v.shape[1], v.double()
    w = ((v - v[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(n, device=x.device)
    keep = (k <= 0) | (rank < k)
    w = torch.where(keep, w, 0.0)
    before = w.cumsum(-1) - w
    keep = keep & ((p >= 1) | (before < p * w.sum(-1, keepdim=True))) & (w >= m) & ((t > 0) | (rank == 0))
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    total = w.cumsum(-1)
    past = total > s["u"].double()[:, None] * total[:, -1:]
    token = past.int().argmax(-1, keepdim=True)
    # the probability with which it was drawn
    return {"tokens": token[:, 0], "logprobs": (w.gather(1, token) / total[:, -1:]).log()[:, 0].float()}


def _plan_own(s):
    c = s["case"]
    positions, slots, q_starts, kv_lens, taken = _qlinear().plan_step(
        s["page_table"], s["lengths"], s["new_tokens"], page_size=c["page"], max_tokens=s["max_tokens"],
        free_pages=s["free_pages"], taken=s["taken"])
    return {"positions": positions, "slots": slots, "q_starts": q_starts, "kv_lens": kv_lens, "taken": taken,
            "page_table": s["page_table"]}


def _plan_plain(s):
    ps, have, new = s["case"]["page"], s["lengths"].long(), s["new_tokens"].long()
    kv = have + new
    held, needed = (have + ps - 1) // ps, (kv + ps - 1) // ps
    ends, fresh = new.cumsum(0), (needed - held).cumsum(0)
    col = torch.arange(s["page_table"].shape[1], device="cuda")[None]
    source = s["taken"] + (fresh - (needed - held))[:, None] + col - held[:, None]
    grown = s["free_pages"][source.clamp(0, s["free_pages"].shape[0] - 1)]
    table = torch.where((col >= held[:, None]) & (col < needed[:, None]), grown, s["page_table"])
    s["page_table"].copy_(table)
    t = torch.arange(s["max_tokens"], device="cuda")
    owner = torch.searchsorted(ends, t, right=True)
    real = owner < new.shape[0]
    owner = owner.clamp(max=new.shape[0] - 1)
    at = torch.where(real, kv[owner] - ends[owner] + t, 0)
    slots = torch.where(real, table[owner, at // ps].long() * ps + at % ps, -1)
    starts = torch.cat([ends.new_zeros(1), ends])
    return {"positions": at, "slots": slots, "q_starts": starts.int(), "kv_lens": kv.int(), "taken": (s["taken"] + fresh[-1:]).int(),
            "page_table": s["page_table"]}


def _sinks_own(s):
    c = s["case"]
    o = _qlinear().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["q_starts"], s["kv_lens"],
                                   max_q=s["max_q"], max_kv=s["max_kv"], window=c["window"], sinks=c["sinks"])
    return {"o": o}


def _plain_width(c):
    """Positions of a sequence that the plain form gathers: the first tokens and what some new token's window holds."""
    q, kv = _lens(c)
    return min(max(kv), c["sinks"] + c["window"] + max(q) - 1)


def _sinks_plain(s):
    """The first tokens and the window's positions of each sequence gathered, all padded to the longest, one softmax."""
    c = s["case"]
    b, ps, hkv, d, sinks, window = c["batch"], c["page"], c["hkv"], c["d"], c["sinks"], c["window"]
    g, n, m = c["hq"] // hkv, _plain_width(c), s["max_q"]
    q_lens = s["q_starts"][1:] - s["q_starts"][:-1]
    kv = s["kv_lens"][:, None].long()
    j = torch.arange(n, device="cuda")[None]
    # positions: j itself, from the end of the first tokens on moved up to the window of the first new token
    shift = (kv - q_lens[:, None] + 1 - window - sinks).clamp(min=0)
    pos = torch.where(j < sinks, j, j + shift)
    at = pos.clamp(max=s["page_table"].shape[1] * ps - 1)
    page = s["page_table"].long().gather(1, at // ps).clamp(min=0)
    k = s["k_cache"][page, :, at % ps].transpose(1, 2).float()
    v = s["v_cache"][page, :, at % ps].transpose(1, 2).float()
    i = torch.arange(m, device="cuda")
    rows = (s["q_starts"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(b, m, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * m, d)
    x = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hkv, g, m, n)
    own_at = (kv - q_lens[:, None] + i)[..., None]
    pos = pos[:, None]
    seen = (pos <= own_at) & (pos < kv[..., None]) & ((pos > own_at - window) | (pos < sinks))
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(b, hkv, g * m, n) @ v).view(b, hkv, g, m, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, m, c["hq"], d)
    return {"o": o[i < q_lens[:, None]].to(s["q"].dtype)}


_own = {"sample": _sample_own, "plan": _plan_own, "sinks": _sinks_own}
_plain = {"sample": _sample_plain, "plan": _plan_plain, "sinks": _sinks_plain}


# ----------------------------------------------------------------------------- the definition, in 64 bits

def _exact_token(x, u, t, k, p, m):
    """One row: a walk down the order of the logits, then up the order of the indices."""
    order = torch.argsort(x, descending=True, stable=True)
    if t == 0:
        return int(order[0]), 0.0
    w = torch.exp((x - x.max()) / t)[order]
    if k > 0:
        w = w[:k]
    if p < 1:
        sums = torch.cumsum(w, 0)
        w = w[:1 + int((sums < p * sums[-1]).sum())]
    w = w[:max(1, int((w >= m).sum()))]
    index, back = torch.sort(order[:w.shape[0]])
    sums = torch.cumsum(w[back], 0)
    at = min(int((sums <= u * sums[-1]).sum()), w.shape[0] - 1)
    return int(index[at]), math.log(float(w[back[at]]) / float(sums[-1]))


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    if c["op"] == "sample":
        u = s["u"].double().tolist()
        each = [s[k].double().tolist() if isinstance(s[k], torch.Tensor) else [s[k]] * c["rows"]
                for k in ("temperature", "top_k", "top_p", "min_p")]
        out = [_exact_token(s["logits"][b].double(), u[b], each[0][b], int(each[1][b]), each[2][b], each[3][b]) for b in range(c["rows"])]
        return {"tokens": torch.tensor([a for a, _ in out], device="cuda"),
                "logprobs": torch.tensor([a for _, a in out], dtype=torch.float64, device="cuda")}
    if c["op"] == "plan":
        ps, table, free = c["page"], s["page_table"].tolist(), s["free_pages"].tolist()
        taken = s["taken"].tolist()[0]
        positions, slots, starts, lens = [], [], [0], []
        for b, (h, n) in enumerate(zip(s["lengths"].tolist(), s["new_tokens"].tolist())):
            for at in range(h, h + n):
                if at % ps == 0:
                    table[b][at // ps] = free[taken]
                    taken += 1
                positions.append(at)
                slots.append(table[b][at // ps] * ps + at % ps)
            starts.append(len(positions))
            lens.append(h + n)
        pad = s["max_tokens"] - len(positions)

        def whole(x, dtype):
            return torch.tensor(x, dtype=dtype, device="cuda")

        return {"positions": whole(positions + [0] * pad, torch.int64), "slots": whole(slots + [-1] * pad, torch.int64),
                "q_starts": whole(starts, torch.int32), "kv_lens": whole(lens, torch.int32), "taken": whole([taken], torch.int32),
                "page_table": whole(table, torch.int32)}
    q, kv = _lens(c)
    out = torch.zeros(sum(q), c["hq"], c["d"], dtype=torch.float64, device="cuda")
    g, at = c["hq"] // c["hkv"], 0
    for b in range(c["batch"]):
        first = max(0, kv[b] - q[b] + 1 - c["window"])
        j = torch.cat([torch.arange(min(c["sinks"], first), device="cuda"), torch.arange(first, kv[b], device="cuda")])
        pages = s["page_table"][b].long()[j // c["page"]]
        i = kv[b] - q[b] + torch.arange(q[b], device="cuda")[:, None]
        hide = (j > i) | ((i - j >= c["window"]) & (j >= c["sinks"]))
        for h in range(c["hkv"]):
            k = s["k_cache"][pages, h, j % c["page"]].double()
            v = s["v_cache"][pages, h, j % c["page"]].double()
            for e in range(h * g, h * g + g):
                x = s["q"][at:at + q[b], e].double() @ k.T / c["d"] ** 0.5
                out[at:at + q[b], e] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
        at += q[b]
    return {"o": out}
