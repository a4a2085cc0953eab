"""Measured cases of the decoder-side operators: rotary append to a paged key/value cache, attention for
a batch of sequences that share a long prefix, and the residual RMS norm with 16-bit or 8-bit output.

They are what a program runs after a search: the retrieved text is the shared prefix (or the candidates
are the sequences), and a decoder reads it to rerank or to answer.  ``own`` selects the framework's
kernels; otherwise the operators run in their plain form, elementary torch operations in 32 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
E4M3_MAX = 448.0
SCALE_FLOOR = 1e-12  # of a row or group whose values are all zero
# (query heads, key/value heads, head dim): the framework's encoder heads, the same shared by threes, and
# generic decoder layouts (groups of 4, 7, 8 and one key/value head for all)
HEADS = [(12, 12, 64), (12, 4, 64), (32, 8, 128), (28, 4, 128), (16, 2, 128), (8, 1, 64), (16, 16, 128)]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one short conversation, one new token: latency
        dict(name="append-1tok", op="append", dtype="bf16", q_heads=12, kv_heads=12, head_dim=64, page=16, seqs=1,
             q_lo=1, q_hi=1, past_lo=77, past_hi=77, prefix=0, rot=64, interleaved=False, lens=1),
        # 100 retrieved chunks of U[64, 512] tokens appended behind one query, the rerank batch
        dict(name="append-rerank", op="append", dtype="f16", q_heads=32, kv_heads=8, head_dim=128, page=64, seqs=100,
             q_lo=64, q_hi=512, past_lo=0, past_hi=0, prefix=333, rot=128, interleaved=False, lens=2),
        # a decoding step of 256 answers, partial rotation of neighbouring pairs
        dict(name="append-decode256", op="append", dtype="bf16", q_heads=28, kv_heads=4, head_dim=128, page=32, seqs=256,
             q_lo=1, q_hi=1, past_lo=0, past_hi=1023, prefix=4096, rot=64, interleaved=True, lens=3),
        # four answers over a short context: latency
        dict(name="attend-decode4", op="attend", dtype="f16", q_heads=12, kv_heads=4, head_dim=64, page=16, seqs=4,
             q_lo=1, q_hi=1, past_lo=0, past_hi=40, prefix=333, lens=4),
        # 64 answers over one retrieved context
        dict(name="attend-decode64", op="attend", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, seqs=64,
             q_lo=1, q_hi=1, past_lo=0, past_hi=511, prefix=4096, lens=5),
        # 256 answers over a very long context
        dict(name="attend-decode256", op="attend", dtype="bf16", q_heads=28, kv_heads=4, head_dim=128, page=32, seqs=256,
             q_lo=1, q_hi=1, past_lo=0, past_hi=1023, prefix=32768, lens=6),
        # eight unrelated long conversations, nothing shared
        dict(name="attend-long8", op="attend", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=128, seqs=8,
             q_lo=1, q_hi=1, past_lo=3000, past_hi=60000, prefix=0, lens=7),
        # the rerank batch: 100 chunks of U[64, 512] tokens read behind one instruction and query
        dict(name="attend-rerank", op="attend", dtype="f16", q_heads=32, kv_heads=8, head_dim=128, page=64, seqs=100,
             q_lo=64, q_hi=512, past_lo=0, past_hi=0, prefix=333, lens=2),
        # reading a long context once, to share it later
        dict(name="attend-prompt", op="attend", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, seqs=1,
             q_lo=8192, q_hi=8192, past_lo=0, past_hi=0, prefix=0, lens=8),
        # one token's row: latency
        dict(name="norm-1row", op="norm", dtype="bf16", rows=1, hidden=768, out8=False, group=0),
        # a decoding step's rows for an 8-bit product, one scale a row; an odd width
        dict(name="norm-256x4095-8bit", op="norm", dtype="f16", rows=256, hidden=4095, out8=True, group=0),
        # a rerank batch's rows for an 8-bit product, one scale for 128 values
        dict(name="norm-28800-8bit", op="norm", dtype="bf16", rows=28800, hidden=4096, out8=True, group=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """The larger of the plain form's padded scores and the operator's own pairs, and the cached elements."""
    n, past = _lengths(c)
    own_len = max(a + b for a, b in zip(n, past))
    padded = c["seqs"] * max(n) * c["q_heads"] * (c["prefix"] + own_len)
    cached = sum(a + b for a, b in zip(n, past)) * c["kv_heads"] * c["head_dim"]
    return padded, cached, c["seqs"] * own_len * c["kv_heads"] * c["head_dim"]


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "norm"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "norm":
        hidden = rng.choice([384, 768, 2048, 4096, 5120, 8192, _log(rng, 33, 8191) | 1])
        rows = _log(rng, 1, max(2, min(28800, 28800 * 4096 // hidden)))
        out8 = rng.random() < 0.5
        return dict(op=op, dtype=dtype, rows=rows, hidden=hidden, out8=out8,
                    group=128 if out8 and hidden % 128 == 0 and rng.random() < 0.5 else 0)
    while True:
        hq, hkv, d = rng.choice(HEADS)
        kind = rng.choice(["decode", "decode", "extend", "prompt"])
        if kind == "decode":
            q_lo = q_hi = 1
            seqs = _log(rng, 1, 256)
            past_lo, past_hi = sorted((_log(rng, 1, 8192) - 1, _log(rng, 1, 8192) - 1))
            prefix = rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 32768)])
        elif kind == "extend":
            seqs = _log(rng, 2, 128)
            q_lo, q_hi = sorted((_log(rng, 1, 512), _log(rng, 1, 512)))
            past_lo, past_hi = 0, rng.choice([0, _log(rng, 1, 512)])
            prefix = rng.choice([0, _log(rng, 16, 4096)])
        else:
            seqs = rng.choice([1, 1, 2, 4])
            q_lo = q_hi = _log(rng, 513, 8192)
            past_lo, past_hi = 0, 0
            prefix = rng.choice([0, 0, _log(rng, 16, 4096)])
        c = dict(op=op, dtype=dtype, q_heads=hq, kv_heads=hkv, head_dim=d, page=rng.choice([16, 32, 64, 128]),
                 seqs=seqs, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, prefix=prefix,
                 lens=rng.randrange(1 << 20))
        padded, cached, gathered = _cost(c)
        if op == "attend" and padded <= 32 * 8192 * 8192 and cached <= 2 ** 28 and gathered <= 2 ** 29:
            return c
        if op == "append" and sum(_lengths(c)[0]) <= 28800 and cached <= 2 ** 27:
            rot = rng.choice([d, d, d // 2])
            return dict(c, rot=rot, interleaved=rng.random() < 0.3)


def _lengths(c):
    """New tokens and earlier cached tokens of every sequence."""
    r = random.Random(c["lens"])
    n = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"])]
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["seqs"])]
    return n, past


def work(case):
    c = case
    if c["op"] == "norm":
        e = c["rows"] * c["hidden"]
        out = e + 4 * c["rows"] * (c["hidden"] // c["group"] if c["group"] else 1) if c["out8"] else 2 * e
        return {"bytes": 6 * e + out + 4 * c["hidden"], "flops": 5 * e}
    n, past = _lengths(c)
    t, d, hq, hkv = sum(n), c["head_dim"], c["q_heads"], c["kv_heads"]
    if c["op"] == "append":
        table = 4 * c["rot"] * min(t, max(a + b for a, b in zip(n, past)))
        return {"bytes": 4 * t * d * (hq + 2 * hkv) + table, "flops": 3 * t * c["rot"] * (hq + hkv)}
    pairs = sum(a * c["prefix"] + a * b + a * (a + 1) // 2 for a, b in zip(n, past))
    keys = c["prefix"] + sum(n) + sum(past)
    return {"bytes": 4 * keys * hkv * d + 4 * t * hq * d + 4 * t * hq, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ inputs
def _pages(c, n, past, gen):
    """Scattered page numbers: the prefix's, then each sequence's; and how many pages the pool has."""
    ps = c["page"]
    counts = [-(-c["prefix"] // ps)] + [-(-(a + b) // ps) for a, b in zip(n, past)]
    total = sum(counts) + 3
    order = torch.randperm(total, generator=gen).tolist()
    lists, at = [], 0
    for k in counts:
        lists.append(order[at:at + k])
        at += k
    return lists[0], lists[1:], total


def _rope_table(positions, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float32, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float32, device="cuda")[:, None] * inv
    return a.cos().contiguous(), a.sin().contiguous()


def prepare(case, seed):
    c = case
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=dev, device="cuda", dtype=torch.float32) * std).to(dt)

    s = dict(c, seed=seed)
    if c["op"] == "norm":
        rows, hidden = c["rows"], c["hidden"]
        loud = 1.0 + 15.0 * (torch.rand(hidden, generator=dev, device="cuda") < 0.01).float()  # a few loud channels
        s["x"] = randn(rows, hidden)
        s["residual"] = (torch.randn(rows, hidden, generator=dev, device="cuda") * 3.0 * loud).to(dt)
        s["weight"] = 1.0 + 0.2 * torch.randn(hidden, generator=dev, device="cuda")
        s["residual_out"] = torch.empty_like(s["x"])
        return s
    n, past = _lengths(c)
    hq, hkv, d, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    t = sum(n)
    prefix_pages, own_pages, total = _pages(c, n, past, gen)
    s["k_pool"] = torch.empty(total, hkv, ps, d, dtype=dt, device="cuda")
    s["v_pool"] = torch.empty(total, hkv, ps, d, dtype=dt, device="cuda")
    for pool in (s["k_pool"], s["v_pool"]):
        for part in pool.split(4096):
            part.copy_(torch.randn(part.shape, generator=dev, device="cuda", dtype=torch.float32))
    seq = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n))
    start = torch.tensor([0] + n).cumsum(0)
    place = torch.arange(t) - start[seq] + torch.tensor(past)[seq]  # of each new token among its sequence's own
    wide = max(len(p) for p in own_pages)
    table = torch.tensor([p + [0] * (wide - len(p)) for p in own_pages], dtype=torch.int64).reshape(len(n), wide)
    if c["op"] == "append":
        qkv = randn(t, (hq + 2 * hkv) * d)  # as a projection leaves it
        s["q"] = qkv[:, : hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d: (hq + hkv) * d].view(t, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
        s["cos"], s["sin"] = _rope_table(c["prefix"] + max(a + b for a, b in zip(n, past)), c["rot"])
        s["position"] = (place + c["prefix"]).cuda()
        s["page_of"] = table[seq, place // ps].cuda()
        s["slot_of"] = (place % ps).cuda()
        s["q_out"] = torch.empty(t, hq, d, dtype=dt, device="cuda")
    else:
        s["q"] = randn(t, hq, d, std=2.0)
        s["seq"], s["step_of"] = seq.cuda(), (torch.arange(t) - start[seq]).cuda()
        s["n"], s["past"] = torch.tensor(n).cuda(), torch.tensor(past).cuda()
        s["prefix_pages"] = torch.tensor(prefix_pages, dtype=torch.int64).cuda()
        s["table"] = table.cuda()
        s["longest"] = max(n)
        s["out"] = torch.empty(t, hq, d, dtype=dt, device="cuda")
        s["lse"] = torch.empty(t, hq, dtype=torch.float32, device="cuda")
    if own:  # the plan of a step: one for all layers
        from ripvec_b200.decode import DecodeStep, PagedCache

        s["cache"] = PagedCache(s["k_pool"], s["v_pool"])
        s["plan"] = DecodeStep(q_heads=hq, kv_heads=hkv, head_dim=d, page_size=ps, device=0)
        s["plan"].plan(q_lens=n, own_lens=[a + b for a, b in zip(n, past)], own_pages=own_pages,
                       prefix_lens=[c["prefix"]], prefix_pages=[prefix_pages], num_pages=total)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        if s["op"] == "append":
            s["plan"].append(s["cache"], s["q"], s["k"], s["v"], s["cos"], s["sin"], q_out=s["q_out"],
                             interleaved=s["interleaved"])
            return s["q_out"], s["k_pool"], s["v_pool"]
        if s["op"] == "attend":
            s["plan"].attend(s["cache"], s["q"], out=s["out"], lse=s["lse"])
            return s["out"], s["lse"]
        from ripvec_b200.decode import rms_norm

        y, scales = rms_norm(s["x"], s["weight"], residual=s["residual"], residual_out=s["residual_out"], eps=EPS,
                             out_8bit=s["out8"], group=s["group"])
        return (y, s["residual_out"], scales) if s["out8"] else (y, s["residual_out"])
    return {"append": _plain_append, "attend": _plain_attend, "norm": _plain_norm}[s["op"]](s)


def _rotate(x, cos, sin, rot, interleaved):
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    c, s = cos[:, None, :], sin[:, None, :]
    y = torch.stack((a * c - b * s, b * c + a * s), -1 if interleaved else -2).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_append(s):
    cos, sin = s["cos"][s["position"]], s["sin"][s["position"]]
    q = _rotate(s["q"], cos, sin, s["rot"], s["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"], cos, sin, s["rot"], s["interleaved"]).to(s["q"].dtype)
    s["k_pool"][s["page_of"], :, s["slot_of"]] = k
    s["v_pool"][s["page_of"], :, s["slot_of"]] = s["v"]
    return q, s["k_pool"], s["v_pool"]


def _plain_attend(s):
    t, hq, d = s["q"].shape
    hkv, ps, b, longest, prefix = s["kv_heads"], s["page"], s["seqs"], s["longest"], s["prefix"]
    g = hq // hkv
    # queries padded to the longest sequence: [kv head, sequence, query x group, d]
    q = torch.zeros(b, longest, hkv, g, d, dtype=torch.float32, device="cuda")
    q[s["seq"], s["step_of"]] = s["q"].float().view(t, hkv, g, d) / math.sqrt(d)
    q = q.permute(2, 0, 1, 3, 4).reshape(hkv, b, longest * g, d)
    pages = s["table"].shape[1]
    k = s["k_pool"][s["table"]].float().permute(2, 0, 1, 3, 4).reshape(hkv, b, pages * ps, d)
    v = s["v_pool"][s["table"]].float().permute(2, 0, 1, 3, 4).reshape(hkv, b, pages * ps, d)
    at = torch.arange(pages * ps, device="cuda")
    step = torch.arange(longest, device="cuda").repeat_interleave(g)
    seen = at <= (s["past"][:, None] + step)[:, :, None]  # [sequence, query x group, key]
    x = (q @ k.transpose(-1, -2)).masked_fill_(~seen, -math.inf)
    # the shared prefix: all sequences' rows against one copy of its keys
    if prefix:
        kp = s["k_pool"][s["prefix_pages"]].float().permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix]
        vp = s["v_pool"][s["prefix_pages"]].float().permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix]
        xp = (q.reshape(hkv, -1, d) @ kp.transpose(-1, -2)).view(hkv, b, longest * g, prefix)
        m = torch.maximum(x.amax(-1, keepdim=True), xp.amax(-1, keepdim=True))
        x, xp = x.sub_(m).exp_(), xp.sub_(m).exp_()
        total = x.sum(-1, keepdim=True) + xp.sum(-1, keepdim=True)
        y = x @ v + (xp.view(hkv, -1, prefix) @ vp).view(hkv, b, -1, d)
    else:
        m = x.amax(-1, keepdim=True)
        x = x.sub_(m).exp_()
        total = x.sum(-1, keepdim=True)
        y = x @ v
    y = (y / total).view(hkv, b, longest, g, d).permute(1, 2, 0, 3, 4)[s["seq"], s["step_of"]]
    lse = (m + total.log()).view(hkv, b, longest, g).permute(1, 2, 0, 3)[s["seq"], s["step_of"]]
    return y.reshape(t, hq, d).to(s["q"].dtype), lse.reshape(t, hq)


def _plain_norm(s):
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    h = h.to(s["x"].dtype)
    if not s["out8"]:
        return y.to(s["x"].dtype), h
    rows, hidden = y.shape
    y = y.view(rows, -1, s["group"] or hidden)
    scales = y.abs().amax(-1).clamp(min=SCALE_FLOOR) / E4M3_MAX
    codes = (y / scales[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(rows, hidden), h, scales


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "attend": _exact_attend, "norm": _exact_norm}[case["op"]](s)


def _exact_append(s):
    position = s["position"].cpu()
    c, si = s["cos"].double().cpu()[position].cuda(), s["sin"].double().cpu()[position].cuda()
    rot = s["rot"]
    first = torch.arange(rot // 2, device="cuda") * (2 if s["interleaved"] else 1)
    second = first + (1 if s["interleaved"] else rot // 2)

    def turned(x):
        y = x.double().clone()
        for h in range(x.shape[1]):
            y[:, h, first] = x[:, h, first].double() * c - x[:, h, second].double() * si
            y[:, h, second] = x[:, h, first].double() * si + x[:, h, second].double() * c
        return y

    k, v = s["k_pool"].double(), s["v_pool"].double()
    kt = turned(s["k"])
    for h in range(s["kv_heads"]):
        k[s["page_of"], h, s["slot_of"]] = kt[:, h]
        v[s["page_of"], h, s["slot_of"]] = s["v"][:, h].double()
    return turned(s["q"]), k, v


def _exact_attend(s):
    n, past = _lengths(s)
    t, hq, d = s["q"].shape
    hkv, prefix = s["kv_heads"], s["prefix"]
    g = hq // hkv
    out = torch.empty(t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(t, hq, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (a, p) in enumerate(zip(n, past)):
        own_pages = s["table"][b][: -(-(a + p) // s["page"])]
        for h in range(hkv):
            kv = [torch.cat((pool[s["prefix_pages"], h].reshape(-1, d)[:prefix], pool[own_pages, h].reshape(-1, d)[: a + p])).double()
                  for pool in (s["k_pool"], s["v_pool"])]
            x = torch.einsum("igd,kd->gik", s["q"][t0:t0 + a, h * g:(h + 1) * g].double(), kv[0]) * d ** -0.5
            hidden = torch.arange(prefix + a + p, device="cuda")[None, :] > prefix + p + torch.arange(a, device="cuda")[:, None]
            x.masked_fill_(hidden, -math.inf)
            l = torch.logsumexp(x, -1)
            lse[t0:t0 + a, h * g:(h + 1) * g] = l.T
            out[t0:t0 + a, h * g:(h + 1) * g] = torch.einsum("gik,kd->igd", (x - l[..., None]).exp_(), kv[1])
        t0 += a
    return out, lse


def _exact_norm(s):
    h = s["x"].double() + s["residual"].double()
    y = s["weight"].double() * h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[1] + EPS)
    if not s["out8"]:
        return y, h
    parts = y.split(s["group"] or y.shape[1], dim=1)
    scales = torch.stack([p.abs().max(1).values for p in parts], 1).clamp(min=SCALE_FLOOR) / E4M3_MAX
    return torch.cat([p / scales[:, i:i + 1] for i, p in enumerate(parts)], 1), h, scales
