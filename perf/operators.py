"""Workloads of the paged serving operators: the 4-bit key/value cache and
attention over it, the norm and rotation of queries and keys, the page tables
and slot maps, and the verification of drafted tokens.

``run`` computes each in elementary torch operations, or, where ``own`` is
true, through rustyllm_b200.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # page tables of a decode step: 16 requests, one new token each
        dict(name="pages-decode", op="pages", batch=16, new="one", top=4096, page=16),
        # page tables of a step that takes in prompts: 200 requests, some of them decoding
        dict(name="pages-prompts", op="pages", batch=200, new="prompt", top=613, page=64),
        # q/k norm and rotation of a decode step: 5 requests of a 64/8-head model, the framework's f32 activations
        dict(name="rope-decode", op="rope", tokens=5, heads=64, kv=8, dim=128, rot=128, type="f32", norm=True, inter=False),
        # the same of a long prompt inside one packed bf16 qkv matrix
        dict(name="rope-prompt", op="rope", tokens=8191, heads=64, kv=8, dim=128, rot=128, type="bf16", norm=True, inter=False),
        # append of a decode step: 64 requests
        dict(name="append-decode", op="append", tokens=64, kv=8, dim=128, type="f32", page=16),
        # append of a long prompt
        dict(name="append-prompt", op="append", tokens=16001, kv=8, dim=128, type="bf16", page=64),
        # one request's decode step, where latency counts
        dict(name="attn-one", op="attn", batch=1, heads=64, kv=8, dim=128, type="f32", queries=1, keys=2000, even=True, page=16, window=0),
        # a batch's decode step, lengths of all kinds
        dict(name="attn-batch", op="attn", batch=64, heads=32, kv=8, dim=128, type="bf16", queries=1, keys=8192, even=False, page=16, window=0),
        # one request's decode step on a very long cache
        dict(name="attn-long", op="attn", batch=1, heads=64, kv=8, dim=128, type="f32", queries=1, keys=131072, even=True, page=64, window=0),
        # prompts' chunks on top of cached ones
        dict(name="attn-prompts", op="attn", batch=3, heads=64, kv=8, dim=128, type="bf16", queries=512, keys=4500, even=False, page=32, window=0),
        # verification of one request's four drafted tokens
        dict(name="verify-one", op="verify", batch=1, drafts=4, vocab=32000, type="f32", point=False),
        # verification of a batch's, over a large vocabulary
        dict(name="verify-batch", op="verify", batch=32, drafts=7, vocab=128003, type="f32", point=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    tops = {}
    for c in listed():
        w = work(c)
        t = tops.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in t:
            t[k] = max(t[k], w[k])
    op = rng.choice(["pages", "rope", "append", "attn", "attn", "verify"])
    heads, kv = rng.choice([(8, 2), (8, 8), (12, 12), (14, 2), (16, 1), (24, 8), (28, 4), (32, 8), (64, 8)])
    dim = rng.choice([32, 64, 64, 96, 128, 128])
    kind = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 16, 32, 64, 128])
    while True:
        if op == "pages":
            new = rng.choice(["one", "prompt"])
            c = dict(op=op, batch=_log(rng, 1, 200), new=new, top=_log(rng, 3, 4096 if new == "one" else 613), page=page)
        elif op == "rope":
            rot = rng.choice([dim, dim, dim // 2])
            c = dict(op=op, tokens=_log(rng, 1, 8191), heads=heads, kv=kv, dim=dim, rot=rot, type=kind, norm=rng.random() < 0.7, inter=rng.random() < 0.3)
        elif op == "append":
            c = dict(op=op, tokens=_log(rng, 1, 16001), kv=kv, dim=dim, type=kind, page=page)
        elif op == "attn":
            queries = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 512)])
            c = dict(op=op, batch=_log(rng, 1, 64), heads=heads, kv=kv, dim=dim, type=kind, queries=queries, keys=_log(rng, queries, 131072), even=rng.random() < 0.3,
                     page=page, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
        else:
            c = dict(op=op, batch=_log(rng, 1, 32), drafts=rng.randint(0, 8), vocab=_log(rng, 200, 128003), type=kind, point=rng.random() < 0.2)
        w = work(c)
        if all(w[k] <= tops[op][k] for k in w) and (op != "attn" or c["batch"] * c["keys"] * kv * dim <= 64 * 8192 * 8 * 128 and
                                                     c["batch"] * c["keys"] * c["queries"] * heads <= 3 * 4500 * 512 * 64):
            return c


# ------------------------------------------------------------------ inputs

def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _spread(lo, hi, n, g):
    """n lengths from lo to hi in an order of the generator's, with one sum whatever the order."""
    every = torch.linspace(hi, lo, n, device=DEV, dtype=torch.float64).round().to(torch.int32)
    return every[torch.randperm(n, device=DEV, generator=g)]


def _lengths(case, g):
    """The keys of each request (the new ones among them) and its queries."""
    b, keys, queries = case["batch"], case["keys"], case["queries"]
    if case["even"]:
        n_q = torch.full((b,), queries, device=DEV, dtype=torch.int32)
        n_k = torch.full((b,), keys, device=DEV, dtype=torch.int32)
    else:
        n_q = _spread(max(1, queries // 2), queries, b, g)
        n_k = torch.randint(queries, keys + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
        n_k[-1] = keys
    return n_k, n_q


def _pool(case, g, rows, heads):
    """Keys and values of `rows` slots with the outlier channels that keys have, drawn in the type that they are appended in."""
    wide = 1.0 + 4.0 * (torch.rand(heads, case["dim"], device=DEV, generator=g) > 0.95)
    k = (_rand(g, rows, heads, case["dim"]) * wide).to(TYPES[case["type"]])
    v = (_rand(g, rows, heads, case["dim"]) * 0.5).to(TYPES[case["type"]])
    return k, v


def _plain_codes(x):
    """Blocks of 32: the f16 scale and the 4-bit codes, two to a byte."""
    blocks = x.float().unflatten(-1, (-1, 32))
    at = blocks.abs().argmax(-1, keepdim=True)
    d = (blocks.gather(-1, at) / -8.0).clamp(-65504.0, 65504.0).half()
    wide = d.double()
    codes = torch.floor(blocks.double() / torch.where(wide == 0, 1.0, wide) + 8.5).clamp(0, 15)
    codes = torch.where(wide == 0, 8.0, codes).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), d.squeeze(-1)


def _plain_values(codes, d):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (c.unflatten(-1, (-1, 32)) * d.float().unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    return _prepare(case, seed, own)


def _prepare(case, seed, ours):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] in ("append", "attn"):
        return (_prepare_append if case["op"] == "append" else _prepare_attn)(case, g, ours)
    return {"pages": _prepare_pages, "rope": _prepare_rope, "verify": _prepare_verify}[case["op"]](case, g)


def _prepare_pages(case, g):
    b, page, top = case["batch"], case["page"], case["top"]
    new = torch.ones(b, device=DEV, dtype=torch.int32)
    if case["new"] == "prompt":
        # seven in ten take in a prompt
        new[:max(1, b * 7 // 10)] = _spread(1, top, max(1, b * 7 // 10), g)
        new = new[torch.randperm(b, device=DEV, generator=g)]
    ctx = torch.randint(0, top + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    width = 2 * top // page + 2
    held = (ctx + page - 1) // page
    n_pages = b * width
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    # the pages that the requests hold come first in `order`, those of the free ring after them
    first = held.cumsum(0) - held
    col = torch.arange(width, device=DEV)
    table = torch.where(col < held[:, None], order[(first[:, None] + col).clamp(max=n_pages - 1).long()], -1).to(torch.int32).contiguous()
    taken = int(held.sum())
    ring = torch.cat((order[taken:], order[:taken])).contiguous()
    head = int(torch.randint(0, n_pages, (1,), device=DEV, generator=g))
    ring = ring.roll(head)
    free = torch.tensor([head, n_pages - taken, 0], device=DEV, dtype=torch.int32)
    # room for the largest sum of new tokens, rounded up as a captured graph's would be
    tokens = b if case["new"] == "one" else (int(new.sum()) + 255) // 256 * 256
    return dict(case=case, ctx=ctx, new=new, table=table, ring=ring, free=free, tokens=tokens, page=page)


def _prepare_rope(case, g):
    n, h, kv, dim, rot = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"]
    # q, k and v side by side, as one product leaves them
    qkv = _rand(g, n, h + 2 * kv, dim).to(TYPES[case["type"]])
    top = max(8192, n)
    freq = 500000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * freq
    pos = torch.randint(0, top, (n,), device=DEV, generator=g, dtype=torch.int32)
    qw = (1.0 + 0.1 * _rand(g, dim)) if case["norm"] else None
    kw = (1.0 + 0.1 * _rand(g, dim)) if case["norm"] else None
    return dict(case=case, q=qkv[:, :h], k=qkv[:, h:h + kv], cos=angle.cos().float(), sin=angle.sin().float(), pos=pos, qw=qw, kw=kw, eps=1e-6)


def _prepare_append(case, g, ours):
    n, kv, dim, page = case["tokens"], case["kv"], case["dim"], case["page"]
    k, v = _pool(case, g, n, kv)
    pages = (n + page - 1) // page + 2
    slots = torch.randperm(pages * page, device=DEV, generator=g)[:n].to(torch.int32)
    s = dict(case=case, k=k, v=v, slots=slots, every=torch.arange(pages * page, device=DEV, dtype=torch.int32))
    if ours:
        from rustyllm_b200.kv4 import KV4Cache
        s["cache"] = KV4Cache(pages, page, kv, dim)
    else:
        for name in "kv":
            s[name + "_codes"] = torch.full((pages * page, kv, dim // 2), 0x88, device=DEV, dtype=torch.uint8)
            s[name + "_d"] = torch.zeros(pages * page, kv, dim // 32, device=DEV, dtype=torch.float16)
    return s


def _prepare_attn(case, g, ours):
    b, h, kv, dim, page, t = case["batch"], case["heads"], case["kv"], case["dim"], case["page"], TYPES[case["type"]]
    n_k, n_q = _lengths(case, g)
    width = (case["keys"] + page - 1) // page
    pages = b * width + 3
    table = torch.randperm(pages, device=DEV, generator=g)[:b * width].reshape(b, width).to(torch.int32).contiguous()
    cu = torch.zeros(b + 1, device=DEV, dtype=torch.int32)
    cu[1:] = n_q.cumsum(0)
    q = _rand(g, int(cu[-1]), h, dim).to(t)
    s = dict(case=case, q=q, table=table, n_k=n_k, n_q=n_q, cu=cu, page=page, scale=dim ** -0.5)
    rows, part = pages * page, max(page, (1 << 26) // (kv * dim) // page * page)
    if ours:
        from rustyllm_b200.kv4 import KV4Cache
        s["cache"] = KV4Cache(pages, page, kv, dim)
    else:
        for name in "kv":
            s[name + "_codes"] = torch.empty(rows, kv, dim // 2, device=DEV, dtype=torch.uint8)
            s[name + "_d"] = torch.empty(rows, kv, dim // 32, device=DEV, dtype=torch.float16)
    for at in range(0, rows, part):
        end = min(rows, at + part)
        k, v = _pool(case, g, end - at, kv)
        if ours:
            s["cache"].append(k, v, torch.arange(at, end, device=DEV, dtype=torch.int32))
        else:
            for name, x in (("k", k), ("v", v)):
                s[name + "_codes"][at:end], s[name + "_d"][at:end] = _plain_codes(x)
    return s


def _prepare_verify(case, g):
    b, n, vocab, t = case["batch"], case["drafts"], case["vocab"], TYPES[case["type"]]
    logits = 3.0 * _rand(g, b, n + 1, vocab)
    p = torch.softmax(logits, -1).to(t)
    q = torch.softmax(logits[:, :n] + 0.7 * _rand(g, b, n, vocab), -1)
    drafts = torch.multinomial(q.reshape(b * n, vocab), 1, generator=g).reshape(b, n).to(torch.int32) if n else torch.zeros(b, 0, device=DEV, dtype=torch.int32)
    counts = torch.randint(max(0, n - 3), n + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    return dict(case=case, p=p, q=None if case["point"] else q.to(t), drafts=drafts, counts=counts, u=torch.rand(b, n, device=DEV, generator=g), r=torch.rand(b, device=DEV, generator=g))


# --------------------------------------------------------------------- run

def run(s):
    return {"pages": _run_pages, "rope": _run_rope, "append": _run_append, "attn": _run_attn, "verify": _run_verify}[s["case"]["op"]](s)


def _run_pages(s):
    if own:
        from rustyllm_b200.pages import pages_extend
        r = pages_extend(s["ctx"], s["new"], s["table"], s["ring"], s["free"], s["page"], s["tokens"])
        return dict(table=s["table"], free=r.free, kv_lens=r.kv_lens, cu=r.cu_new, positions=r.positions, slots=r.slots)
    ctx, new, table, page = s["ctx"].long(), s["new"].long(), s["table"], s["page"]
    held = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - held
    first = need.cumsum(0) - need
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    at = (s["free"][0] + first[:, None] + col - held[:, None]) % s["ring"].numel()
    full = torch.where(fresh, s["ring"][at], table)
    cu = torch.zeros(new.numel() + 1, device=DEV, dtype=torch.int64)
    cu[1:] = new.cumsum(0)
    token = torch.arange(s["tokens"], device=DEV)
    row = torch.searchsorted(cu[1:], token, right=True).clamp(max=new.numel() - 1)
    live = token < cu[-1]
    pos = torch.where(live, ctx[row] + token - cu[row], -1)
    slot = torch.where(live, full[row, (pos // page).clamp(min=0)].long() * page + pos % page, -1)
    taken = need.sum()
    free = torch.stack(((s["free"][0] + taken) % s["ring"].numel(), s["free"][1] - taken, torch.zeros_like(taken)))
    i32 = torch.int32
    return dict(table=full.to(i32), free=free.to(i32), kv_lens=(ctx + new).to(i32), cu=cu.to(i32), positions=pos.to(i32), slots=slot.to(i32))


def _plain_rope(x, w, s):
    case = s["case"]
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * w
    rot = case["rot"]
    c, n = s["cos"][s["pos"].long()].unsqueeze(1), s["sin"][s["pos"].long()].unsqueeze(1)
    turned, rest = y[..., :rot], y[..., rot:]
    if case["inter"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * c - b * n, a * n + b * c), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _run_rope(s):
    if own:
        from rustyllm_b200.rope import qk_norm_rope
        q, k = qk_norm_rope(s["q"], s["k"], s["pos"], s["cos"], s["sin"], q_weight=s["qw"], k_weight=s["kw"], eps=s["eps"], interleaved=s["case"]["inter"])
        return dict(q=q, k=k)
    return dict(q=_plain_rope(s["q"], s["qw"], s), k=_plain_rope(s["k"], s["kw"], s))


def _run_append(s):
    if own:
        s["cache"].append(s["k"], s["v"], s["slots"])
        k, v = s["cache"].read(s["every"])
        return dict(k=k, v=v)
    out, slots = {}, s["slots"].long()
    for name in "kv":
        s[name + "_codes"][slots], s[name + "_d"][slots] = _plain_codes(s[name])
        out[name] = _plain_values(s[name + "_codes"][s["every"].long()], s[name + "_d"][s["every"].long()])
    return out


def _run_attn(s):
    case = s["case"]
    if own:
        one = case["queries"] == 1
        return s["cache"].attention(s["q"], s["table"], s["n_k"], cu_q=None if one else s["cu"], max_q=case["queries"], scale=s["scale"], window=case["window"],
                                    max_len=case["keys"])
    b, h, kv, dim, keys, most = case["batch"], case["heads"], case["kv"], case["dim"], case["keys"], case["queries"]
    slots = (s["table"].long()[:, :, None] * s["page"] + torch.arange(s["page"], device=DEV)).flatten(1)[:, :keys]
    k = _plain_values(s["k_codes"][slots], s["k_d"][slots]).permute(0, 2, 3, 1)  # [b, kv, dim, keys]
    v = _plain_values(s["v_codes"][slots], s["v_d"][slots]).transpose(1, 2)      # [b, kv, keys, dim]
    i = torch.arange(most, device=DEV)
    row = (s["cu"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    live = i < s["n_q"][:, None]
    q = s["q"].float()[row].unflatten(2, (kv, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, queries * group, dim]
    p = (q @ k).mul_(s["scale"]).unflatten(2, (most, h // kv))
    j = torch.arange(keys, device=DEV)
    pos = (s["n_k"] - s["n_q"])[:, None, None] + i[None, :, None]
    seen = (j <= pos) & live[:, :, None]
    if case["window"]:
        seen &= j > pos - case["window"]
    p.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (most, h // kv)) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, queries, heads, dim]
    return o[live].to(s["q"].dtype)


def _run_verify(s):
    if own:
        from rustyllm_b200.spec import spec_verify
        tokens, accepted = spec_verify(s["p"], s["drafts"], s["u"], s["r"], q=s["q"], n_drafts=s["counts"])
        return dict(tokens=tokens, accepted=accepted)
    p, q, drafts = s["p"], s["q"], s["drafts"].long()
    b, n = drafts.shape
    at = torch.arange(n + 1, device=DEV)
    px = p[:, :n].gather(2, drafts[..., None]).squeeze(2).double()
    qx = q.gather(2, drafts[..., None]).squeeze(2).double() if q is not None else torch.ones_like(px)
    good = (s["u"].double() * qx < px) & (at[:n] < s["counts"][:, None])
    accepted = good.long().cumprod(1).sum(1)
    each = torch.arange(b, device=DEV)
    left = p[each, accepted].double()
    if n:
        rejected = accepted < s["counts"]
        which = accepted.clamp(max=n - 1)
        if q is not None:
            less = (left - q[each, which].double()).clamp(min=0)
        else:
            less = left.scatter(1, drafts[each, which][:, None], 0.0)
        less = torch.where(less.sum(1, keepdim=True) > 0, less, left)
        left = torch.where(rejected[:, None], less, left)
    upto = left.cumsum(1)
    last = (left > 0).long().mul(torch.arange(1, left.shape[1] + 1, device=DEV)).amax(1) - 1
    token = torch.minimum((upto <= s["r"].double()[:, None] * upto[:, -1:]).sum(1), last)
    shown = torch.cat((drafts, torch.zeros(b, 1, device=DEV, dtype=torch.int64)), 1)
    tokens = torch.where(at < accepted[:, None], shown, torch.where(at == accepted[:, None], token[:, None], -1))
    return dict(tokens=tokens.to(torch.int32), accepted=accepted.to(torch.int32))


# -------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "pages":
        tokens = case["batch"] if case["new"] == "one" else int(case["batch"] * (0.35 * case["top"] + 0.65))
        # lengths in, lengths and offsets out, half the table and the new pages; a position and a slot for each token
        return {"bytes": case["batch"] * 20 + tokens * (8 + 8 / case["page"]), "flops": tokens * 4}
    if op == "rope":
        n = case["tokens"] * (case["heads"] + case["kv"]) * case["dim"]
        return {"bytes": 2 * n * SIZE[case["type"]] + case["tokens"] * (4 + 4 * case["rot"]), "flops": n * 10}
    if op == "append":
        page = case["page"]
        every = ((case["tokens"] + page - 1) // page + 2) * page
        n, m = case["tokens"] * 2 * case["kv"] * case["dim"], every * 2 * case["kv"] * case["dim"]
        return {"bytes": n * (SIZE[case["type"]] + 4.5 / 8) + m * (4 + 4.5 / 8), "flops": n * 6}
    if op == "attn":
        share = 1.0 if case["even"] else 0.5
        seqs = case["batch"] * share + (1 - share)
        queries = case["batch"] * case["queries"] if case["even"] else 0.75 * case["batch"] * case["queries"] if case["queries"] > 1 else case["batch"]
        keys = min(case["keys"], case["window"] + case["queries"]) if case["window"] else case["keys"]
        seen = max(1.0, keys * share - case["queries"] / 2)
        if case["window"]:
            seen = min(seen, case["window"])
        per = case["kv"] * case["dim"] * 2 * 4.5 / 8
        return {"bytes": seqs * keys * per + 2 * queries * case["heads"] * case["dim"] * SIZE[case["type"]],
                "flops": 4.0 * queries * case["heads"] * case["dim"] * seen}
    rows = case["batch"] * case["vocab"] * SIZE[case["type"]]
    return {"bytes": rows * (1 if case["point"] else 2) + case["batch"] * case["drafts"] * 16, "flops": 3 * case["batch"] * case["vocab"]}


# ------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits, request by request."""
    s = _prepare(case, seed, False)
    op = case["op"]
    if op == "rope":
        rot, half = case["rot"], case["rot"] // 2
        phase = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None, :]
        out = {}
        for name, w in (("q", s["qw"]), ("k", s["kw"])):
            x = s[name].double()
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt() * w.double()
            first = torch.arange(0, rot, 2, device=DEV) if case["inter"] else torch.arange(half, device=DEV)
            second = first + (1 if case["inter"] else half)
            z = torch.complex(x[..., first], x[..., second]) * phase
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[name] = y
        return out
    if op == "append":
        out = {}
        for name in "kv":
            blocks = s[name].double().unflatten(-1, (-1, 32))
            big, small = blocks.amax(-1, keepdim=True), blocks.amin(-1, keepdim=True)
            size = torch.maximum(big, -small)
            # of two elements of one size and both signs the first decides
            signed = torch.where(big > -small, big, small)
            both = (big == -small) & (size > 0)
            first = torch.where((blocks == big).int().argmax(-1, keepdim=True) < (blocks == small).int().argmax(-1, keepdim=True), big, small)
            d = (torch.where(both, first, signed) / -8).clamp(-65504, 65504).half().double()
            levels = torch.arange(-8, 8, device=DEV, dtype=torch.float64)
            # the nearest level, the higher code of two that are as near
            code = ((blocks / torch.where(d == 0, 1.0, d)).unsqueeze(-1) >= levels[1:] - 0.5).sum(-1)
            values = torch.where(d == 0, 0.0, levels[code] * d).flatten(-2)
            whole = torch.zeros(s["every"].numel(), *values.shape[1:], device=DEV, dtype=torch.float64)
            whole[s["slots"].long()] = values
            out[name] = whole
        return out
    if op == "attn":
        out = torch.empty(s["q"].shape, device=DEV, dtype=torch.float64)
        h, kv, group = case["heads"], case["kv"], case["heads"] // case["kv"]
        n_k, cu = s["n_k"].tolist(), s["cu"].tolist()
        for b in range(case["batch"]):
            j = torch.arange(n_k[b], device=DEV)
            slots = s["table"][b].long()[j // s["page"]] * s["page"] + j % s["page"]
            i = torch.arange(cu[b + 1] - cu[b], device=DEV)
            pos = n_k[b] - i.numel() + i
            hidden = (j[None] > pos[:, None]) | ((j[None] <= pos[:, None] - case["window"]) if case["window"] else False)
            for x in range(kv):
                values = []
                for name in "kv":
                    codes, d = s[name + "_codes"][slots, x], s[name + "_d"][slots, x]
                    c = torch.empty(n_k[b], case["dim"], device=DEV, dtype=torch.float64)
                    c[:, 0::2], c[:, 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
                    values.append(c * d.double().repeat_interleave(32, 1))
                for head in range(x * group, (x + 1) * group):
                    score = s["q"][cu[b]:cu[b + 1], head].double() @ values[0].T * case["dim"] ** -0.5
                    weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
                    out[cu[b]:cu[b + 1], head] = weight @ values[1]
        return out
    return None
