"""The serving operators over a paged key/value cache, as work to measure.

Four operators, which a server with many streams runs one after another:

* append:  the step's rotated keys and its values go into the pages of their
  sequences, the rotated queries come out (with a norm of each query and key
  head where the model has one)
* attention:  ragged batches of queries over the pages (decode and prompt chunks)
* tree:  the same for a tree of drafted tokens, whose ancestors a bit mask names
* sample:  a token for each row of logits, from given random numbers

`run` computes them in plain torch, or calls `hetero_infer_b200.ops` where
`own` is true.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- cases -------------------------------------------------------------------
# rows: new tokens of a sequence, from rows_lo to rows_hi; ctx: entries that the
# cache holds before them; `shape` seeds the lengths, which belong to the case.

def _append(name, **kw):
    c = dict(op="append", act="bf16", cache="bf16", heads=28, kv=4, hd=128, page=16, seqs=1, rows_lo=1, rows_hi=1,
             ctx_lo=0, ctx_hi=0, norm=False, tree=False, shape=1)
    return {"name": name, **c, **kw}


def _attn(name, op="attention", **kw):
    c = dict(op=op, act="bf16", cache="bf16", heads=28, kv=4, hd=128, page=16, seqs=1, rows_lo=1, rows_hi=1, ctx_lo=0,
             ctx_hi=0, shape=1)
    return {"name": name, **c, **kw}


def _sample(name, **kw):
    c = dict(op="sample", act="f32", rows=1, vocab=152064, peaks=40)
    return {"name": name, **c, **kw}


def listed():
    return [
        # one decode step of eight streams (the pipeline's microbatches), fp32 projections into an fp16 cache
        _append("append_decode_8", act="f32", cache="f16", seqs=8, ctx_lo=32, ctx_hi=2000),
        # one long prompt, chunked by nothing: bandwidth
        _append("append_prompt_8191", seqs=1, rows_lo=8191, rows_hi=8191, page=64),
        # a mixed step of a model that norms its query and key heads: odd rows, narrow heads
        _append("append_norm_ragged", act="f16", cache="f16", heads=32, kv=8, hd=64, seqs=37, rows_lo=1, rows_hi=61,
                ctx_lo=0, ctx_hi=900, norm=True),
        # the end of a 32-token prompt's 128-token answer, one stream: latency
        _attn("decode_1x159", seqs=1, ctx_lo=159, ctx_hi=159),
        # a full decode batch at every age: bandwidth
        _attn("decode_64_ragged", seqs=64, ctx_lo=100, ctx_hi=8200, page=32),
        # one stream with a long cache, fp32 queries
        _attn("decode_1x131071_f32", act="f32", cache="f16", seqs=1, ctx_lo=131071, ctx_hi=131071, page=64),
        # prompt chunks of four streams on what they have already: arithmetic
        _attn("prompt_chunks_4", seqs=4, rows_lo=1025, rows_hi=2048, ctx_lo=0, ctx_hi=4096, page=64),
        # a drafted tree of one stream
        _attn("tree_1x26", op="tree", seqs=1, rows_lo=26, rows_hi=26, ctx_lo=1001, ctx_hi=1001),
        # drafted trees of sixteen streams
        _attn("tree_16x64", op="tree", seqs=16, rows_lo=40, rows_hi=64, ctx_lo=200, ctx_hi=4100, page=32),
        # one stream's token
        _sample("sample_1", rows=1),
        # a batch with parameters of its own for each row
        _sample("sample_64", rows=64),
        # many rows of 16-bit logits (equal values among them), a smaller vocabulary
        _sample("sample_256_bf16", act="bf16", rows=256, vocab=32003),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "tree", "sample"))
    if op == "sample":
        vocab = _span(rng, 300, 152064)
        rows = _span(rng, 1, max(1.0, min(256.0, 9.7e6 / vocab)))
        return {k: v for k, v in _sample("", act=rng.choice(("f32", "f32", "bf16", "f16")), rows=rows, vocab=vocab,
                                         peaks=rng.randint(0, 200)).items() if k != "name"}
    cache = rng.choice(("bf16", "f16"))
    act = rng.choice(("f32", cache, cache))
    kv = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 12))
    hd = rng.choice((32, 64, 64, 96, 128, 128, 128, 192, 256))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    base = dict(act=act, cache=cache, heads=kv * group, kv=kv, hd=hd, page=page, shape=rng.randrange(1 << 20))
    if op == "append":
        seqs = _span(rng, 1, 128)
        top = max(1, min(8191, int(3.5e7 / (kv * (group + 1) * hd) / seqs)))
        hi = _span(rng, 1, top)
        c = _append("", **base, seqs=seqs, rows_lo=rng.randint(1, hi), rows_hi=hi, ctx_lo=0, ctx_hi=_span(rng, 1, 4000),
                    norm=rng.random() < 0.4, tree=rng.random() < 0.3)
    elif op == "tree":
        seqs = _span(rng, 1, 16)
        hi = _span(rng, 2, 100)
        room = 4.5e8 / (seqs * kv * hd * (1 + hi * group / 100))
        c = _attn("", op="tree", **base, seqs=seqs, rows_lo=rng.randint(1, hi), rows_hi=hi, ctx_lo=rng.randint(0, 60),
                  ctx_hi=_span(rng, 61, max(62.0, min(16000.0, room))))
    elif rng.random() < 0.6:  # decode: one row a sequence, or a few
        seqs = _span(rng, 1, 64)
        hi = rng.choice((1, 1, 1, 2, 5))
        room = 1.3e8 / (seqs * kv * hd)
        c = _attn("", **base, seqs=seqs, rows_lo=1, rows_hi=hi, ctx_lo=rng.randint(0, 60),
                  ctx_hi=_span(rng, 61, max(62.0, min(131071.0, room))))
    else:  # prompt chunks
        seqs = _span(rng, 1, 6)
        hi = _span(rng, 16, 2048)
        room = 1.2e11 / (seqs * kv * group * hd * hi) - hi
        c = _attn("", **base, seqs=seqs, rows_lo=rng.randint(1, hi), rows_hi=hi, ctx_lo=0,
                  ctx_hi=_span(rng, 1, max(2.0, min(16000.0, room))))
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(case):
    """(new rows, entries before them) of each sequence."""
    r = random.Random(case["shape"])
    rows = [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    return rows, ctx


def _parents(case, n, s):
    """The parent of each node of sequence s's tree; -1 for one that follows the cache itself."""
    r = random.Random(case["shape"] * 1009 + s)
    return [-1 if i == 0 else r.randint(max(-1, i - 9), i - 1) for i in range(n)]


# ---- inputs ------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)

    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        x = randn(n, v) * 2.0
        if case["peaks"]:  # the few tokens that a trained model holds likely
            at = (rand(n, case["peaks"]) * v).long()
            x.scatter_add_(1, at, 6.0 + 3.0 * randn(n, case["peaks"]))
        f = rand(4, n)
        temperature = torch.where(f[0] < 0.1, torch.zeros_like(f[0]), 0.5 + 0.9 * f[0]).float()
        top_k = torch.where(f[1] < 0.4, torch.zeros_like(f[1]), 1 + 150 * f[1]).int()
        top_p = torch.where(f[2] < 0.3, torch.ones_like(f[2]), 0.6 + 0.39 * f[2]).float()
        min_p = torch.where(f[3] < 0.5, torch.zeros_like(f[3]), 0.1 * f[3]).float()
        return dict(op="sample", logits=x.to(TYPES[case["act"]]), u=rand(n), temperature=temperature, top_k=top_k,
                    top_p=top_p, min_p=min_p)

    act, cache = TYPES[case["act"]], TYPES[case["cache"]]
    H, KV, D, ps = case["heads"], case["kv"], case["hd"], case["page"]
    rows, ctx = _lengths(case)
    total = sum(rows)
    need = [-(-(c + r) // ps) for c, r in zip(ctx, rows)]
    per_seq = max(need)
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    # each sequence's pages in the order that a server under load has them: any; unused places hold -1
    first = [sum(need[:i]) for i in range(len(need))]
    slot = torch.tensor(first, device="cuda")[:, None] + torch.arange(per_seq, device="cuda")
    used = torch.arange(per_seq, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    pages = torch.where(used, order[slot.clamp(max=n_pages - 1)], torch.full_like(order[:1], -1)).contiguous()
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    st = dict(op=case["op"], pages=pages, cu_rows=torch.tensor(cu, dtype=torch.int32, device="cuda"),
              lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"), max_rows=max(rows),
              max_len=max(c + r for c, r in zip(ctx, rows)),
              k_cache=randn(n_pages, KV, ps, D, dtype=cache), v_cache=randn(n_pages, KV, ps, D, dtype=cache))
    if case["op"] == "append":
        qkv = randn(total, (H + 2 * KV) * D, dtype=act)  # one fused projection: q, k and v are views of its rows
        st["q"] = qkv[:, :H * D].view(total, H, D)
        st["k"] = qkv[:, H * D:(H + KV) * D].view(total, KV, D)
        st["v"] = qkv[:, (H + KV) * D:].view(total, KV, D)
        n = st["max_len"]
        inv = 1e6 ** (-torch.arange(0, D // 2, dtype=torch.float64, device="cuda") * 2 / D)
        ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
        st["rope_cos"], st["rope_sin"] = ang.cos().float(), ang.sin().float()
        st["q_norm"] = 1 + 0.1 * randn(D) if case["norm"] else None
        st["k_norm"] = 1 + 0.1 * randn(D) if case["norm"] else None
        st["positions"] = None
        if case["tree"]:  # a node's position is its depth's, not its place in the cache
            pos = []
            for s, (r, c) in enumerate(zip(rows, ctx)):
                depth = []
                for p in _parents(case, r, s):
                    depth.append(0 if p < 0 else depth[p] + 1)
                pos += [c + d for d in depth]
            st["positions"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    else:
        st["q"] = randn(total, H, D, dtype=act) * 1.5
        st["scale"] = D ** -0.5
    if case["op"] == "tree":
        words = (max(rows) + 31) // 32
        mask = []
        for s, r in enumerate(rows):
            seen = []
            for i, p in enumerate(_parents(case, r, s)):
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            for b in seen:
                w = [b >> 32 * j & 0xFFFFFFFF for j in range(words)]
                mask.append([x - (1 << 32) if x >> 31 else x for x in w])
        st["tree_mask"] = torch.tensor(mask, dtype=torch.int32, device="cuda")
    return st


# ---- one pass ------------------------------------------------------------------

def run(s):
    if own:
        from hetero_infer_b200 import ops
        if s["op"] == "append":
            q = ops.paged_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["cu_rows"],
                                 s["lens"], s["rope_cos"], s["rope_sin"], positions=s["positions"],
                                 q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if s["op"] == "attention":
            return {"out": ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["cu_rows"],
                                               s["lens"], scale=s["scale"])}
        if s["op"] == "tree":
            return {"out": ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["cu_rows"], s["lens"],
                                              s["tree_mask"], scale=s["scale"])}
        tok, logp = ops.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                    top_p=s["top_p"], min_p=s["min_p"], logprob=True)
        return {"token": tok, "logprob": logp}
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "sample":
        return _plain_sample(s)
    return _plain_attention(s)


def _row_places(s, n):
    """Of each of n rows: its sequence and its place among that sequence's rows."""
    t = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s["cu_rows"][1:].contiguous(), t, right=True)
    return seq, t - s["cu_rows"][seq]


def _plain_append(s):
    q, k, v = s["q"], s["k"], s["v"]
    D, ps = q.shape[-1], s["k_cache"].shape[2]
    seq, at = _row_places(s, q.shape[0])
    at = s["lens"][seq] + at
    pos = at if s["positions"] is None else s["positions"]
    cos, sin = s["rope_cos"][pos][:, None], s["rope_sin"][pos][:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    page, off = s["pages"][seq, at // ps], at % ps
    s["k_cache"][page, :, off] = turned(k, s["k_norm"]).to(s["k_cache"].dtype)
    s["v_cache"][page, :, off] = v.to(s["v_cache"].dtype)
    return {"q": turned(q, s["q_norm"]).to(q.dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    q, kc, vc, lens = s["q"], s["k_cache"], s["v_cache"], s["lens"]
    n, H, D = q.shape
    KV, ps, S, R, L = kc.shape[1], kc.shape[2], lens.shape[0], s["max_rows"], s["max_len"]
    seq, place = _row_places(s, n)
    count = s["cu_rows"][1:] - s["cu_rows"][:-1]
    at = torch.arange(L, device="cuda")
    r = torch.arange(R, device="cuda")
    page = s["pages"][:, at // ps].clamp(min=0)
    k = kc[page, :, (at % ps)[None].expand(S, L)].float()  # [S, L, KV, D]
    v = vc[page, :, (at % ps)[None].expand(S, L)].float()
    row = (s["cu_rows"][:-1, None] + r).clamp(max=n - 1)
    x = q[row].float().view(S, R, KV, H // KV, D)
    new = at[None] - lens[:, None]  # an entry's place among the new ones
    if s["op"] == "tree":
        m = s["tree_mask"]
        w = (new >> 5).clamp(0, m.shape[1] - 1)
        bits = m[row].gather(2, w[:, None].expand(S, R, L)) >> (new & 31)[:, None] & 1
        seen = (new < 0)[:, None] | ((bits == 1) & (new < count[:, None])[:, None])
    else:
        seen = new[:, None] <= r[None, :, None]
    seen = seen[:, None, None]
    z = torch.einsum("srkgd,slkd->skgrl", x, k) * s["scale"]
    z = torch.where(seen, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1)
    o = torch.einsum("skgrl,slkd->srkgd", e, v)
    total = total.permute(0, 3, 1, 2)[..., None]
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return {"out": o.reshape(S, R, H, D)[seq, place].to(q.dtype)}


def _plain_sample(s):
    x = s["logits"].double()
    n, v = x.shape
    t = s["temperature"].double()[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    val, idx = torch.sort(x, dim=-1, descending=True, stable=True)  # equal values: the lowest index first
    w = e.gather(1, idx)
    rank = torch.arange(v, device="cuda")
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    before = w.cumsum(-1) - w
    group = torch.ones_like(w, dtype=torch.bool)  # the mass above a value: that before the first of its equals
    group[:, 1:] = val[:, 1:] != val[:, :-1]
    above = torch.where(group, before, torch.full_like(before, -1.0)).cummax(-1).values
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (above < p * w.sum(-1, keepdim=True))
    keep &= w >= s["min_p"].double()[:, None]
    w = torch.where(keep, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, idx, w)
    c = w.cumsum(-1)
    tok = (c <= s["u"][:, None] * c[:, -1:]).sum(-1)
    logp = torch.log(w.gather(1, tok.clamp(max=v - 1)[:, None])[:, 0] / c[:, -1])
    greedy = t[:, 0] <= 0
    tok = torch.where(greedy, idx[:, 0], tok)
    return {"token": tok.int(), "logprob": torch.where(greedy, torch.zeros_like(logp), logp).float()}


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * BYTES[case["act"]] + case["rows"] * 32, "flops": 4 * n}
    rows, ctx = _lengths(case)
    H, KV, D = case["heads"], case["kv"], case["hd"]
    a, c = BYTES[case["act"]], BYTES[case["cache"]]
    if case["op"] == "append":
        n = sum(rows)
        return {"bytes": n * D * ((2 * H + 2 * KV) * a + 2 * KV * c) + n * 4 * D,
                "flops": n * (H + KV) * D * (6 if case["norm"] else 3)}
    entries = sum(r + x for r, x in zip(rows, ctx))
    if case["op"] == "tree":
        pairs = 0
        for s, (r, x) in enumerate(zip(rows, ctx)):
            depth = []
            for p in _parents(case, r, s):
                depth.append(1 if p < 0 else depth[p] + 1)
            pairs += r * x + sum(depth)
    else:
        pairs = sum(r * x + r * (r + 1) // 2 for r, x in zip(rows, ctx))
    return {"bytes": entries * KV * D * 2 * c + sum(rows) * H * D * 2 * a, "flops": 4 * pairs * H * D}


# ---- the definition, in 64 bits ------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    rows, ctx = _lengths(case)
    D, ps = case["hd"], case["page"]
    first = [sum(rows[:i]) for i in range(len(rows))]
    if case["op"] == "append":
        pos = s["positions"].tolist() if s["positions"] is not None else None
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        for i, (r, c) in enumerate(zip(rows, ctx)):
            at = torch.arange(c, c + r, device="cuda")
            where = at if pos is None else torch.tensor(pos[first[i]:first[i] + r], device="cuda")
            # the rotation as a product of complex numbers: (x_j + i x_{j + D/2}) times cos + i sin
            turn = torch.complex(s["rope_cos"][where].double(), s["rope_sin"][where].double())[:, None]
            new = slice(first[i], first[i] + r)
            made = []
            for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
                x = x[new].double()
                if w is not None:
                    x = x * w.double() * (x.square().sum(-1, keepdim=True) / D + 1e-6).rsqrt()
                y = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
                made.append(torch.cat((y.real, y.imag), -1))
            out[new] = made[0]
            page = s["pages"][i].long()[at // ps]
            caches[0][page, :, at % ps] = made[1]
            caches[1][page, :, at % ps] = s["v"][new].double()
        return {"q": out, "k_cache": caches[0], "v_cache": caches[1]}
    H, KV = case["heads"], case["kv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (r, c) in enumerate(zip(rows, ctx)):
        at = torch.arange(c + r, device="cuda")
        page = s["pages"][i].long()[at // ps]
        if case["op"] == "tree":
            hide = torch.ones(r, c + r, dtype=torch.bool)
            hide[:, :c] = False
            par = _parents(case, r, i)
            for j in range(r):
                a = j
                while a >= 0:
                    hide[j, c + a] = False
                    a = par[a]
            hide = hide.cuda()
        for h in range(H):
            k = s["k_cache"][page, h // (H // KV), at % ps].double()
            v = s["v_cache"][page, h // (H // KV), at % ps].double()
            for b in range(0, r, 1024):
                q = s["q"][first[i] + b:first[i] + min(r, b + 1024), h].double()
                z = (q @ k.T) * s["scale"]
                if case["op"] == "tree":
                    z.masked_fill_(hide[b:b + 1024], -math.inf)
                else:
                    z.masked_fill_(at > c + b + torch.arange(q.shape[0], device="cuda")[:, None], -math.inf)
                out[first[i] + b:first[i] + b + q.shape[0], h] = torch.softmax(z, -1) @ v
    return {"out": out}


def _exact_sample(s):
    toks, logps = [], []
    top_k, top_p, min_p = s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist()
    temperature, u = s["temperature"].tolist(), s["u"].tolist()
    for i in range(len(u)):
        x = s["logits"][i].double().cpu()
        if temperature[i] <= 0:
            toks.append(int((x == x.max()).nonzero()[0]))
            logps.append(0.0)
            continue
        p = torch.softmax(x / temperature[i], 0)
        order = torch.argsort(x, descending=True, stable=True)
        kept = order[:top_k[i]] if top_k[i] > 0 else order
        if top_p[i] < 1:
            q = p[kept] / p[kept].sum()
            vals = x[kept]
            c = torch.cumsum(q, 0)
            starts = torch.searchsorted(-vals, -vals, right=False)  # the first of each value's equals
            above = torch.where(starts > 0, c[(starts - 1).clamp(min=0)], torch.zeros_like(c))
            kept = kept[above < top_p[i]]
        kept = kept[p[kept] >= min_p[i] * p.max()]
        kept = kept.sort().values
        c = torch.cumsum(p[kept] / p[kept].sum(), 0)
        j = min(int(torch.searchsorted(c, u[i], right=True)), len(kept) - 1)
        toks.append(int(kept[j]))
        logps.append(float(torch.log(p[kept[j]] / p[kept].sum())))
    return {"token": torch.tensor(toks, dtype=torch.int32), "logprob": torch.tensor(logps, dtype=torch.float64)}
