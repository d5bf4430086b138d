"""The operators of a serving step over a paged key-value cache, as cases that can be timed and compared.

Three operators: appending new tokens' keys and values to a paged cache with the position rotation on the way
("append"), attention of one new token per sequence over that cache ("attention"), and the adjustment of the
logits before sampling: penalties for repeated tokens, biases, grammar masks ("adjust").

`listed` and `draw` give cases (dicts of plain values), `prepare` makes what a program has in hand before the call,
`run` is one pass through the operator, `exact` its result from the definition in 64 bits, `work` what a pass
cannot do without. With `own` false, `run` computes the operator from elementary torch operations; with `own` true
it calls this package.
"""
import math
import random

import torch

own = False


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # -- append: qkv rows of the projection -> normed, rotated q; k and v rows written to their pages
        # one token for one sequence of the 8B model: the smallest decode step, latency alone
        dict(name="append_one", op="append", B=1, T=1, H=32, KV=8, HD=128, page=64, ctx=1000, dtype="f32", norm=True),
        # a decode step of 16 sequences of the 8B model, the engine's largest batch
        dict(name="append_step16", op="append", B=16, T=16, H=32, KV=8, HD=128, page=64, ctx=4096, dtype="f32",
             norm=True),
        # ragged prompts of five sequences, bf16 rows without q/k norm, small heads, odd total
        dict(name="append_ragged", op="append", B=5, T=2503, H=14, KV=2, HD=64, page=16, ctx=700, dtype="bf16",
             norm=False),
        # long prompts appended at far positions: the bandwidth end
        dict(name="append_prompts", op="append", B=4, T=16384, H=32, KV=8, HD=128, page=64, ctx=100000, dtype="f32",
             norm=True),
        # -- attention: one new token per sequence over the paged cache
        # one sequence in the middle of a chat: latency
        dict(name="attend_one", op="attention", B=1, H=32, KV=8, HD=128, page=64, ctx=517, ragged=False, window=0,
             pad=0, dtype="f32", lse=False),
        # the engine's batch of 16 with ragged contexts, two rows of the batch unused
        dict(name="attend_step16", op="attention", B=16, H=32, KV=8, HD=128, page=64, ctx=4096, ragged=True, window=0,
             pad=2, dtype="f32", lse=False),
        # one long document: the cache's length is all there is to split
        dict(name="attend_long", op="attention", B=1, H=32, KV=8, HD=128, page=64, ctx=131072, ragged=False, window=0,
             pad=0, dtype="f32", lse=True),
        # a server's batch of 64 ragged sequences, bf16 rows, small pages: the bandwidth end
        dict(name="attend_serve", op="attention", B=64, H=32, KV=8, HD=128, page=16, ctx=8192, ragged=True, window=0,
             pad=0, dtype="bf16", lse=False),
        # many short sequences with a sliding window, seven small heads to a group
        dict(name="attend_window", op="attention", B=200, H=14, KV=2, HD=64, page=32, ctx=3000, ragged=True,
             window=1024, pad=0, dtype="bf16", lse=True),
        # -- adjust: logits -> adjusted logits (the raw ones are kept for log-probabilities)
        # one chat with repetition and frequency penalties over its last 600 tokens
        dict(name="adjust_one", op="adjust", B=1, V=151936, prior=600, nbias=0, mask=False, dtype="f32"),
        # 16 requests, full rings of prior tokens, some biased tokens, a grammar mask each
        dict(name="adjust_step16", op="adjust", B=16, V=151936, prior=4096, nbias=64, mask=True, dtype="f32"),
        # 256 requests, bf16 logits of an odd vocabulary, everything on: the bandwidth end
        dict(name="adjust_serve", op="adjust", B=256, V=151669, prior=1000, nbias=300, mask=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of its operator."""
    op = rng.choice(["append", "attention", "adjust"])
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        case = _draw_one(rng, op)
        if all(work(case)[k] <= max(w[k] for w in most) for k in ("bytes", "flops")):
            return case


def _draw_one(rng, op):
    if op == "adjust":
        V = rng.choice([1000, 4096, 32000, 50257, 128256, 151669, 151936, _log_int(rng, 500, 200000)])
        B = _log_int(rng, 1, 512)
        return dict(op=op, B=B, V=V, prior=rng.choice([0, 1, _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)]),
                    nbias=rng.choice([0, 1, _log_int(rng, 1, 300)]), mask=rng.random() < 0.6,
                    dtype=rng.choice(["f32", "f32", "bf16"]))
    HD = rng.choice([64, 128, 128])
    KV = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    dtype = rng.choice(["f32", "bf16"])
    if op == "append":
        T = _log_int(rng, 1, 16384)
        B = _log_int(rng, 1, min(T, 256))
        return dict(op=op, B=B, T=T, H=KV * G, KV=KV, HD=HD, page=page, ctx=_log_int(rng, 1, 200000), dtype=dtype,
                    norm=rng.random() < 0.6)
    B = _log_int(rng, 1, 256)
    ctx = _log_int(rng, 1, 131072)
    return dict(op=op, B=B, H=KV * G, KV=KV, HD=HD, page=page, ctx=ctx, ragged=rng.random() < 0.7,
                window=rng.choice([0, 0, _log_int(rng, 1, 4096)]), pad=rng.choice([0, 0, B // 8]), dtype=dtype,
                lse=rng.random() < 0.5)


def _shape_rng(case):
    """Lengths belong to the case, not to a seed: `work` counts them."""
    return random.Random(",".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))


def _append_lengths(case):
    """(new tokens, first position) of every sequence."""
    rng, B, T = _shape_rng(case), case["B"], case["T"]
    cuts = sorted(rng.sample(range(1, T), B - 1)) if B > 1 else []
    new = [b - a for a, b in zip([0] + cuts, cuts + [T])]
    first = [rng.randint(0, case["ctx"]) for _ in range(B)]
    return new, first


def _attention_positions(case):
    """Position of every sequence's new token, -1 in the unused rows of the batch."""
    rng, B, ctx = _shape_rng(case), case["B"], case["ctx"]
    pos = [(rng.randint(1, ctx) if case["ragged"] else ctx) - 1 for _ in range(B)]
    for b in rng.sample(range(B), case["pad"]):
        pos[b] = -1
    return pos


def _span(p, window):
    """Attended positions [lo, hi) of a new token at position p."""
    return (max(0, p - window + 1) if window else 0), p + 1


def _dtype(case):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[case["dtype"]]


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    B = case["B"]
    if case["op"] == "append":
        T, H, KV, HD = case["T"], case["H"], case["KV"], case["HD"]
        rows = T * (2 * H + 2 * KV) * HD * es + T * 2 * KV * HD * 2
        return {"bytes": rows + 4 * (T // case["page"] + B) + 16 * B, "flops": T * (H + KV) * HD * 7}
    if case["op"] == "attention":
        H, KV, HD = case["H"], case["KV"], case["HD"]
        n = 0
        for p in _attention_positions(case):
            lo, hi = _span(p, case["window"])
            n += hi - lo
        io = 2 * B * H * HD * es + (4 * B * H if case["lse"] else 0) + 8 * B + 4 * (n // case["page"])
        return {"bytes": n * KV * HD * 4 + io, "flops": 4 * n * H * HD + 4 * n * H}
    V = case["V"]
    side = 4 * B * case["prior"] + 8 * B * case["nbias"] + (4 * B * ((V + 31) // 32) if case["mask"] else 0) + 12 * B
    return {"bytes": 2 * B * V * es + side, "flops": 5 * B * case["prior"] + B * case["nbias"] + B * V}


# ---------------------------------------------------------------------------------------------- prepare
def _tables(lens, page, gen):
    """Page tables [B, max] (int32) of a pool whose pages are handed out in random order, and the pool's size."""
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    k = 0
    for b, n in enumerate(need):
        table[b, :n] = order[k:k + n]
        k += n
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, B = _dtype(case), case["B"]
    randn = lambda *s, dtype=dt: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    st = dict(case=case)
    if case["op"] == "append":
        T, H, KV, HD, page = case["T"], case["H"], case["KV"], case["HD"], case["page"]
        new, first = _append_lengths(case)
        # a token's page is known by its index in the sequence: pages before the first written one are never
        # touched, so the pool holds the written range only and the entries before it point at page 0
        skip = [f // page for f in first]
        part, pages = _tables([f + n - s * page for f, n, s in zip(first, new, skip)], page, gen)
        width = max(s + part.shape[1] for s in skip)
        table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
        for b, s in enumerate(skip):
            table[b, s:s + part.shape[1]] = part[b]
        cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        st.update(qkv=randn(T, (H + 2 * KV) * HD) * 2, kc=randn(pages, KV, page, HD, dtype=torch.bfloat16),
                  vc=randn(pages, KV, page, HD, dtype=torch.bfloat16), table=table, cu=cu,
                  pos=torch.tensor(first, dtype=torch.int64, device="cuda"), q_out=torch.empty(T, H, HD, dtype=dt,
                                                                                              device="cuda"),
                  inv=1.0 / (1e6 ** (torch.arange(0, HD, 2, dtype=torch.float32, device="cuda") / HD)),
                  qn=None, kn=None, one=T == B)
        if case["norm"]:
            st["qn"] = (1 + 0.1 * randn(HD, dtype=torch.float32)).bfloat16()
            st["kn"] = (1 + 0.1 * randn(HD, dtype=torch.float32)).bfloat16()
        if own:
            from ai_b200 import paged
            st["cache"] = paged.Cache(st["kc"], st["vc"])
    elif case["op"] == "attention":
        H, KV, HD, page = case["H"], case["KV"], case["HD"], case["page"]
        pos = _attention_positions(case)
        table, pages = _tables([p + 1 for p in pos], page, gen)
        st.update(q=randn(B, H, HD) * 1.5, kc=randn(pages, KV, page, HD, dtype=torch.bfloat16),
                  vc=randn(pages, KV, page, HD, dtype=torch.bfloat16), table=table, host_pos=pos,
                  pos=torch.tensor(pos, dtype=torch.int64, device="cuda"),
                  out=torch.empty(B, H, HD, dtype=dt, device="cuda"),
                  lse=torch.empty(B, H, dtype=torch.float32, device="cuda") if case["lse"] else None)
        if own:
            from ai_b200 import paged
            st["cache"] = paged.Cache(st["kc"], st["vc"])
            st["ws"] = paged.workspace(B, H, st["cache"])
    else:
        V = case["V"]
        rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
        st.update(logits=randn(B, V) * 4, out=torch.empty(B, V, dtype=dt, device="cuda"), prior=None, bias_ids=None,
                  bias=None, mask=None, repetition=0.9 + 0.5 * rand(B), presence=rand(B) - 0.25,
                  frequency=0.5 * rand(B) - 0.1)
        if case["prior"]:
            # frequent tokens come many times; the tail of a ring that is not full is -1
            ids = (V * rand(B, case["prior"]) ** 4).to(torch.int32).clamp_(max=V - 1)
            fill = (case["prior"] * (0.5 + rand(B, 1))).to(torch.int32)
            at = torch.arange(case["prior"], device="cuda")[None]
            st["prior"] = torch.where(at < fill, ids, torch.full_like(ids, -1))
        if case["nbias"]:
            st["bias_ids"] = (V * rand(B, case["nbias"])).to(torch.int32).clamp_(max=V - 1)
            st["bias"] = 10 * rand(B, case["nbias"]) - 5
        if case["mask"]:
            # every second grammar state allows about half of the vocabulary, the others about a hundredth
            W = (V + 31) // 32
            word = lambda: torch.randint(-2 ** 31, 2 ** 31, (B, W), generator=gen, device="cuda")  # noqa: E731
            m = word()
            rare = m & word() & word() & word() & word() & word() & word()
            sparse = (torch.arange(B, device="cuda") % 2 == 1)[:, None]
            st["mask"] = torch.where(sparse, rare, m).to(torch.int32)
    return st


# -------------------------------------------------------------------------------------------------- run
def run(st):
    return {"append": _run_append, "attention": _run_attention, "adjust": _run_adjust}[st["case"]["op"]](st)


def _run_append(st):
    c = st["case"]
    T, H, KV, HD, page = c["T"], c["H"], c["KV"], c["HD"], c["page"]
    q, k, v = (t.view(T, -1, HD) for t in st["qkv"].split([H * HD, KV * HD, KV * HD], 1))
    if own:
        from ai_b200 import paged
        paged.append(st["cache"], st["table"], st["pos"], k, v, cu=None if st["one"] else st["cu"], q=q,
                     q_out=st["q_out"], qn=st["qn"], kn=st["kn"], inv=st["inv"], eps=1e-6)
        return st["q_out"], st["kc"], st["vc"]
    t = torch.arange(T, device="cuda")
    seq = (t[:, None] >= st["cu"][None, 1:]).sum(1)
    pos = st["pos"][seq] + t - st["cu"][seq]
    ang = pos[:, None].double() * st["inv"].double()
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    st["q_out"].copy_(rotated(q, st["qn"]))
    at = st["table"][seq, pos // page].long()
    st["kc"][at, :, pos % page] = rotated(k, st["kn"]).bfloat16()
    st["vc"][at, :, pos % page] = v.bfloat16()
    return st["q_out"], st["kc"], st["vc"]


def _run_attention(st):
    c = st["case"]
    H, KV, HD, page = c["H"], c["KV"], c["HD"], c["page"]
    if own:
        from ai_b200 import paged
        paged.attention(st["q"], st["cache"], st["table"], st["pos"], out=st["out"], window=c["window"],
                        lse=st["lse"], ws=st["ws"])
        return st["out"] if st["lse"] is None else (st["out"], st["lse"])
    for b, p in enumerate(st["host_pos"]):
        lo, hi = _span(p, c["window"])
        if hi == lo:
            st["out"][b] = 0
            if st["lse"] is not None:
                st["lse"][b] = -math.inf
            continue
        at = st["table"][b, lo // page:-(-hi // page)].long()
        cut = slice(lo % page, lo % page + hi - lo)
        k = st["kc"][at].transpose(0, 1).reshape(KV, -1, HD)[:, cut].float()
        v = st["vc"][at].transpose(0, 1).reshape(KV, -1, HD)[:, cut].float()
        s = st["q"][b].float().view(KV, H // KV, HD) @ k.transpose(1, 2) * HD ** -0.5
        m = s.amax(-1, keepdim=True)
        e = (s - m).exp()
        z = e.sum(-1, keepdim=True)
        st["out"][b] = ((e @ v) / z).view(H, HD)
        if st["lse"] is not None:
            st["lse"][b] = (m + z.log()).view(H)
    return st["out"] if st["lse"] is None else (st["out"], st["lse"])


def _run_adjust(st):
    c = st["case"]
    B, V = c["B"], c["V"]
    if own:
        from ai_b200 import sampler
        return sampler.adjust(st["logits"], out=st["out"], prior=st["prior"], repetition=st["repetition"],
                              presence=st["presence"], frequency=st["frequency"], bias_ids=st["bias_ids"],
                              bias=st["bias"], mask=st["mask"])
    x = st["logits"].float()
    if st["prior"] is not None:
        ids = st["prior"].long()
        ok = (ids >= 0) & (ids < V)
        n = torch.zeros(B, V, device="cuda").scatter_add_(1, ids.clamp(0, V - 1), ok.float())
        r, p, f = (st[k][:, None] for k in ("repetition", "presence", "frequency"))
        x = torch.where(n > 0, torch.where(x < 0, x * r, x / r) - (n * f + p), x)
    if st["bias"] is not None:
        x = x + torch.zeros(B, V, dtype=torch.float64, device="cuda").scatter_add_(
            1, st["bias_ids"].long(), st["bias"].double()).float()
    if st["mask"] is not None:
        j = torch.arange(V, device="cuda")
        x = torch.where((st["mask"][:, j // 32] >> (j % 32).int()) & 1 != 0, x, -math.inf)
    st["out"].copy_(x)
    return st["out"]


# ------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "adjust": _exact_adjust}[case["op"]](st, case)


def _exact_append(st, c):
    T, H, KV, HD, page, half = c["T"], c["H"], c["KV"], c["HD"], c["page"], c["HD"] // 2
    rows = st["qkv"].double().view(T, H + 2 * KV, HD)
    kc, vc = st["kc"].double(), st["vc"].double()
    q = torch.empty(T, H, HD, dtype=torch.float64, device="cuda")
    new, first = _append_lengths(c)
    done = 0
    for b, (n, f) in enumerate(zip(new, first)):
        x = rows[done:done + n]
        p = torch.arange(f, f + n, device="cuda")
        turn = torch.polar(torch.ones(1, 1, dtype=torch.float64, device="cuda"),
                           torch.outer(p.double(), st["inv"].double()))[:, None]

        def rotated(y, w):
            if w is not None:
                y = y / ((y ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        q[done:done + n] = rotated(x[:, :H], st["qn"])
        at = st["table"][b].long()[p // page]
        kc[at, :, p % page] = rotated(x[:, H:H + KV], st["kn"])
        vc[at, :, p % page] = x[:, H + KV:]
        done += n
    return q, kc, vc


def _exact_attention(st, c):
    B, H, KV, HD, page = c["B"], c["H"], c["KV"], c["HD"], c["page"]
    out = torch.zeros(B, H, HD, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, p in enumerate(st["host_pos"]):
        lo, hi = _span(p, c["window"])
        if hi <= lo:
            continue
        j = torch.arange(lo, hi, device="cuda")
        at = st["table"][b].long()[j // page]
        for g in range(KV):
            k, v = st["kc"][at, g, j % page].double(), st["vc"][at, g, j % page].double()
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            s = st["q"][b, heads].double() @ k.T / math.sqrt(HD)
            lse[b, heads] = torch.logsumexp(s, 1)
            out[b, heads] = torch.softmax(s, 1) @ v
    return (out, lse) if c["lse"] else out


def _exact_adjust(st, c):
    B, V = c["B"], c["V"]
    out = st["logits"].double()
    words = (V + 31) // 32
    for b in range(B):
        x = out[b]
        if st["prior"] is not None:
            ids = st["prior"][b].long()
            ids, n = torch.unique(ids[(ids >= 0) & (ids < V)], return_counts=True)
            y, r = x[ids], st["repetition"][b].double()
            y = torch.where(y < 0, y * r, y / r)
            x[ids] = y - st["frequency"][b].double() * n - st["presence"][b].double()
        if st["bias"] is not None:
            x.index_add_(0, st["bias_ids"][b].long(), st["bias"][b].double())
        if st["mask"] is not None:
            bits = (st["mask"][b, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
            x[bits.view(words * 32)[:V] == 0] = -math.inf
    return out
