"""Operators of ``kiln_b200.api`` as cases that can be timed and compared with their plain forms.

Kinds, by the ``kind`` of a case:

  sample   a token for each row of logits, drawn with temperature, top-k, top-p and min-p from given random numbers
           (``sample_rows``), and its log probability among what was kept
  shared   paged attention of sequences that share a long prefix (``AttentionPlan``): the blocks of the prefix stand in
           the tables of all of them, what follows is their own
  lora     what low-rank adapters add to a projection's rows, each row with its request's adapter or none
           (``Adapters.apply``)

``own`` chooses between the plain form (elementary torch operations, on tensors alone) and the calls of the package.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16      # tokens in a block of the paged cache


def listed():
    return [
        # One user on an 8B model: a row a step, launch latency counts.
        dict(name="sample_1x128256", kind="sample", rows=1, vocab=128256, mode="user", masked=0.0),
        # A small server, every request with settings of its own, two rows under a grammar's mask; a vocabulary that no vector width divides.
        dict(name="sample_7x50001", kind="sample", rows=7, vocab=50001, mode="user", masked=0.25),
        # The rows of a verify round: 32 requests with 5 drafted tokens each, temperature alone (all of a row counts).
        dict(name="sample_192x128256", kind="sample", rows=192, vocab=128256, mode="plain", masked=0.0),
        # The most rows that a step samples, the largest vocabulary.
        dict(name="sample_512x256000", kind="sample", rows=512, vocab=256000, mode="user", masked=0.0),
        # Four continuations of one short prompt: latency counts.
        dict(name="shared_4x1_512", kind="shared", heads=32, kv_heads=8, head_dim=128, batch=4, groups=1, rows=1, prefix=512, lo=3, hi=60, softcap=0.0),
        # Answers sampled about two long documents, 64 of each; heads of 64 features, no length a multiple of a block.
        dict(name="shared_128x1_6001_2", kind="shared", heads=32, kv_heads=8, head_dim=64, batch=128, groups=2, rows=1, prefix=6001, lo=1, hi=333, softcap=0.0),
        # Heads of 256 features under a soft cap, a verify round of four rows.
        dict(name="shared_16x4_6144", kind="shared", heads=16, kv_heads=8, head_dim=256, batch=16, groups=1, rows=4, prefix=6144, lo=20, hi=500, softcap=50.0),
        # The widest layers, 64 requests over a long document, a verify round of five rows each.
        dict(name="shared_64x5_4096", kind="shared", heads=64, kv_heads=8, head_dim=128, batch=64, groups=1, rows=5, prefix=4096, lo=64, hi=512, softcap=0.0),
        # One user with an adapter: a row of a square projection.
        dict(name="lora_1_4096x4096_r16", kind="lora", rows=1, n_in=4096, n_out=4096, rank=16, adapters=1, bare=0.0),
        # A full server in decode, an adapter a request, into the widest projection.
        dict(name="lora_32_4096x28672_r16", kind="lora", rows=32, n_in=4096, n_out=28672, rank=16, adapters=32, bare=0.0),
        # A mixed step: some requests have no adapter; no size a multiple of a tile.
        dict(name="lora_333_3584x11000_r24", kind="lora", rows=333, n_in=3584, n_out=11000, rank=24, adapters=5, bare=0.3),
        # A piece of eight prompts.
        dict(name="lora_2048_4096x28672_r64", kind="lora", rows=2048, n_in=4096, n_out=28672, rank=64, adapters=8, bare=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd ones as likely as even ones."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["sample", "shared", "lora"])
    if kind == "sample":
        vocab = rng.choice([128256, 152064, 256000, _spread(rng, 1000, 256000), _spread(rng, 32000, 256000)])
        return dict(kind=kind, rows=_spread(rng, 1, 512), vocab=vocab, mode=rng.choice(["user", "user", "plain"]), masked=rng.choice([0.0, 0.0, 0.3]))
    most = work([c for c in listed() if c["kind"] == kind][-1])
    while True:
        if kind == "lora":
            rows = _spread(rng, 1, 2048)
            case = dict(kind=kind, rows=rows, n_in=rng.choice([2048, 3584, 4096, 8192, 14336]), n_out=_spread(rng, 500, 28672),
                        rank=rng.choice([8, 16, 16, 32, 64, _spread(rng, 1, 128)]), adapters=_spread(rng, 1, min(rows, 40)), bare=rng.choice([0.0, 0.0, 0.3]))
        else:
            heads, kv_heads, head_dim, softcap = rng.choice([(32, 8, 128, 0.0), (28, 4, 128, 0.0), (32, 8, 64, 0.0), (16, 8, 256, 50.0), (64, 8, 128, 0.0)])
            batch, hi = _spread(rng, 2, 128), _spread(rng, 1, 700)
            case = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, groups=rng.randint(1, min(3, batch // 2)),
                        rows=rng.choice([1, 1, 2, 3, 5, 6]), prefix=_spread(rng, 400, 8192), lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, softcap=softcap)
        if all(work(case)[n] <= most[n] for n in most):
            return case


# ---- what a program has in hand -----------------------------------------------------------------------------------

_context = None


def _ctx():
    """The process's one context: a program opens one for each GPU and keeps it, with its torch work on the context's stream."""
    global _context
    if _context is None:
        from kiln_b200 import api
        _context = api.Context(0)
        torch.cuda.set_stream(torch.cuda.ExternalStream(_context.stream))
    return _context


def _generators(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g, np.random.default_rng([int(seed), salt])


def _sample_inputs(case, seed):
    """Logits as a language model's last layer gives them: most near each other, a few far above; and a setting a row."""
    g, rng = _generators(seed, 1)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty(rows, vocab, device="cuda").normal_(0.0, 2.2, generator=g)
    likely = torch.randint(0, vocab, (rows, 24), device="cuda", generator=g)
    lift = torch.empty(rows, 24, device="cuda").exponential_(0.4, generator=g) + 6.0
    logits.scatter_add_(1, likely, lift)
    masked = int(round(case["masked"] * rows))
    if masked:   # a grammar that allows one token in a hundred
        shut = torch.rand(masked, vocab, device="cuda", generator=g) > 0.01
        shut[:, 0] = False
        logits[:masked][shut] = -math.inf
    logits = logits.to(torch.bfloat16)
    temperature = rng.choice([0.6, 0.7, 0.8, 1.0, 1.0, 1.3], rows).astype(np.float32)
    top_k, top_p, min_p = np.zeros(rows, np.int32), np.ones(rows, np.float32), np.zeros(rows, np.float32)
    if case["mode"] == "user":
        temperature[rng.random(rows) < 0.1] = 0.0
        top_k = rng.choice([0, 0, 20, 40, 64, 1000], rows).astype(np.int32)
        top_p = rng.choice([1.0, 1.0, 0.8, 0.9, 0.95], rows).astype(np.float32)
        min_p = rng.choice([0.0, 0.0, 0.02, 0.05, 0.1], rows).astype(np.float32)
    u = torch.rand(rows, device="cuda", generator=g)
    return logits, temperature, top_k, top_p, min_p, u


def _shared_inputs(case, seed):
    """Pools of K and V [2, blocks, kv heads, BLOCK, features], queries, and a length and a table of blocks a sequence."""
    g, rng = _generators(seed, 2)
    batch, rows, prefix = case["batch"], case["rows"], case["prefix"]
    tails = rng.integers(case["lo"], case["hi"] + 1, batch)
    tails[0], tails[-1] = case["lo"], case["hi"]
    full = prefix // BLOCK                                     # the rest of the prefix is copied, with the sequence's own
    need = [-(-(prefix + int(t) + rows) // BLOCK) - full for t in tails]
    total = case["groups"] * full + sum(need)
    order = rng.permutation(total)                             # a running server's free list is in no order
    heads_of = [order[i * full: (i + 1) * full] for i in range(case["groups"])]
    at, tables = case["groups"] * full, []
    for i, n in enumerate(need):
        tables.append(np.concatenate([heads_of[i * case["groups"] // batch], order[at: at + n]]).astype(np.uint32))
        at += n
    pool = torch.empty(2, total, case["kv_heads"], BLOCK, case["head_dim"], device="cuda").normal_(generator=g).to(torch.bfloat16)
    q = torch.empty(batch * rows, case["heads"], case["head_dim"], device="cuda").normal_(0.0, 1.5, generator=g).to(torch.bfloat16)
    return pool, q, [prefix + int(t) for t in tails], tables


def _lora_inputs(case, seed):
    """Activations, a projection's rows, A [adapters, rank, in], B [adapters, out, rank], a factor an adapter, an adapter a row (-1: none)."""
    g, rng = _generators(seed, 3)
    rows, adapters, rank = case["rows"], case["adapters"], case["rank"]

    def normal(std, *shape):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(torch.bfloat16)
    x, y = normal(1.0, rows, case["n_in"]), normal(1.0, rows, case["n_out"])
    a, b = normal(case["n_in"] ** -0.5, adapters, rank, case["n_in"]), normal(0.05, adapters, case["n_out"], rank)
    scale = rng.choice([0.5, 1.0, 2.0], adapters).astype(np.float32)
    cuts = np.sort(rng.choice(np.arange(1, rows), adapters - 1, replace=False))       # a request's rows stand together
    slots = np.searchsorted(cuts, np.arange(rows), side="right")
    slots = rng.permutation(adapters)[slots]
    slots = np.where(np.isin(slots, np.flatnonzero(rng.random(adapters) < case["bare"])), -1, slots)
    return x, y, a, b, scale, slots.astype(np.int32)


def prepare(case, seed):
    state = dict(case)
    if case["kind"] == "lora":
        x, y, a, b, scale, slots = _lora_inputs(case, seed)
        if own:
            from kiln_b200 import api
            bank = api.Adapters(_ctx(), case["n_in"], case["n_out"], slots=case["adapters"], max_rank=case["rank"])
            for i in range(case["adapters"]):
                bank.set(i, a[i], b[i], float(scale[i]))
            state.update(bank=bank, who=api.AdapterRows(_ctx(), slots), x=x, y=y)
        else:
            state.update(x=x, y=y, a=a, b=b, scale=[float(v) for v in scale],
                         who=[(int(i), torch.from_numpy(np.flatnonzero(slots == i)).cuda()) for i in np.unique(slots) if i >= 0])
        torch.cuda.synchronize()
        return state
    if case["kind"] == "sample":
        logits, temperature, top_k, top_p, min_p, u = _sample_inputs(case, seed)
        if own:
            from kiln_b200 import api
            _ctx()
            settings = [api.SamplingParams(float(t), int(k), float(p), float(m)) for t, k, p, m in zip(temperature, top_k, top_p, min_p)]
            state.update(api=api, logits=logits, params=api.pack_sampling(settings, logits.device), u=u)
        else:
            state.update(logits=logits, u=u, **{n: torch.from_numpy(v).cuda() for n, v in
                                                dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).items()})
        torch.cuda.synchronize()
        return state
    pool, q, lens, tables = _shared_inputs(case, seed)
    scale = case["head_dim"] ** -0.5
    if own:
        from kiln_b200 import api
        ctx = _ctx()
        _, total, kv_heads, _, dim = pool.shape
        kv = api.PagedKv(ctx, api.KvSpec(1, kv_heads, dim, total, BLOCK))
        still = torch.zeros(dim // 2, device="cuda")           # no rotation: the rows are written as they are
        for b in range(0, total, 512):
            k, v = (t[b: b + 512].transpose(1, 2).reshape(-1, kv_heads * dim) for t in pool)
            seq = api.SeqStep(k.shape[0], 0, 0, np.arange(b, b + k.shape[0] // BLOCK, dtype=np.uint32))
            api.rope_kv_write(ctx, kv, 0, torch.cat([k, k, v], 1), still, kv_heads, [seq])
        seqs = [api.SeqStep(case["rows"], n, 0, t) for n, t in zip(lens, tables)]
        state.update(kv=kv, plan=api.AttentionPlan(ctx, kv, case["heads"], seqs), q=q, scale=scale)
    else:
        state.update(pool=pool, q=q, lens=lens, tables=[torch.from_numpy(t.astype(np.int64)).cuda() for t in tables], scale=scale)
    torch.cuda.synchronize()
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------

def _sample_plain(s):
    l = s["logits"].float() + 0.0                              # -0 is +0
    l = torch.where(l.isnan(), -math.inf, l)
    l, index = torch.sort(l, dim=1, descending=True, stable=True)
    top, vocab = l[:, :1], l.shape[1]
    far = torch.where(l == top, 0.0, l - top).double()
    w = torch.where(l == -math.inf, 0.0, torch.exp(far / s["temperature"].double().clamp_min(1e-300)[:, None]))
    cum = torch.cumsum(w, 1)
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < vocab), s["top_k"].long(), vocab)[:, None]
    reach = s["top_p"].double()[:, None] * cum.gather(1, k - 1)
    n = torch.where(s["top_p"][:, None] < 1, (cum < reach).sum(1, keepdim=True) + 1, vocab)
    n = torch.minimum(torch.minimum(n, k), (w >= s["min_p"].double()[:, None]).sum(1, keepdim=True)).clamp(1, vocab)
    mass = cum.gather(1, n - 1)
    j = torch.minimum((cum <= s["u"].double()[:, None] * mass).sum(1, keepdim=True), n - 1)
    greedy = s["temperature"][:, None] <= 0
    j = torch.where(greedy, 0, j)
    logprob = torch.where(greedy, 0.0, torch.log(w.gather(1, j) / mass))
    return index.gather(1, j)[:, 0].int(), logprob[:, 0].float()


def _shared_plain(s):
    pool, q = s["pool"], s["q"].float()
    rows, per = s["rows"], s["heads"] // s["kv_heads"]
    out = torch.empty_like(s["q"])
    for i, (n, table) in enumerate(zip(s["lens"], s["tables"])):
        k, v = (t[table].transpose(1, 2).reshape(-1, s["kv_heads"], s["head_dim"])[: n + rows].float() for t in pool)
        x = q[i * rows: (i + 1) * rows].reshape(rows, s["kv_heads"], per, -1)
        scores = torch.einsum("rhgd,khd->hrgk", x, k) * s["scale"]
        if s["softcap"]:
            scores = s["softcap"] * torch.tanh(scores / s["softcap"])
        seen = torch.arange(n + rows, device=q.device) <= n + torch.arange(rows, device=q.device)[:, None]
        scores = torch.where(seen[None, :, None], scores, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.einsum("hrgk,khd->rhgd", p, v) / p.sum(-1).permute(1, 0, 2)[..., None]
        out[i * rows: (i + 1) * rows] = o.reshape(rows, s["heads"], -1).to(out.dtype)
    return out.reshape(out.shape[0], -1)


def _lora_plain(s):
    out = s["y"].clone()
    for i, rows in s["who"]:
        t = s["x"][rows].float() @ s["a"][i].float().T
        out[rows] = (s["y"][rows].float() + s["scale"][i] * (t @ s["b"][i].float().T)).to(out.dtype)
    return out


def run(state):
    if state["kind"] == "lora":
        return state["bank"].apply(state["x"], state["who"], state["y"]) if own else _lora_plain(state)
    if state["kind"] == "sample":
        return state["api"].sample_rows(_context, state["logits"], state["params"], state["u"]) if own else _sample_plain(state)
    return state["plan"].run(0, state["q"], state["scale"], state["softcap"]) if own else _shared_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "lora":                                 # every row taken to have an adapter
        m, k, n, r = case["rows"], case["n_in"], case["n_out"], case["rank"]
        return {"bytes": 2.0 * (m * k + 2 * m * n + case["adapters"] * r * (k + n)), "flops": 2.0 * m * r * (k + n)}
    if case["kind"] == "sample":                               # the row once; settings, number, token and probability
        return {"bytes": case["rows"] * (2.0 * case["vocab"] + 28), "flops": 2.0 * case["rows"] * case["vocab"]}
    tail, rows = (case["lo"] + case["hi"]) / 2 + case["rows"], case["batch"] * case["rows"]
    keys = case["groups"] * case["prefix"] + case["batch"] * tail
    q = rows * case["heads"] * case["head_dim"]
    return {"bytes": 4.0 * keys * case["kv_heads"] * case["head_dim"] + 4.0 * q, "flops": 4.0 * q * (case["prefix"] + tail)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "lora":
        x, y, a, b, scale, slots = _lora_inputs(case, seed)
        out = y.double()
        for i, slot in enumerate(slots):
            if slot >= 0 and (i == 0 or slots[i - 1] != slot):
                end = i + int(np.argmin(np.append(slots[i:] == slot, False)))
                out[i:end] += (b[slot].double() @ (a[slot].double() @ x[i:end].double().T)).T * float(scale[slot])
        return out
    if case["kind"] == "sample":
        if case["rows"] * case["vocab"] > 50_000_000:
            return None
        logits, temperature, top_k, top_p, min_p, u = _sample_inputs(case, seed)
        logits, u = logits.float().cpu().numpy().astype(np.float64), u.cpu().numpy().astype(np.float64)
        tokens, logprobs = np.zeros(case["rows"], np.int32), np.zeros(case["rows"])
        for r, row in enumerate(logits):
            order = np.argsort(-row, kind="stable")
            if temperature[r] <= 0:
                tokens[r] = order[0]
                continue
            with np.errstate(under="ignore"):
                w = np.exp((row[order] - row[order[0]]) / np.float64(temperature[r]))
            kept = w[: top_k[r]] if top_k[r] > 0 else w
            if top_p[r] < 1:
                sums = np.cumsum(kept)
                kept = kept[: np.searchsorted(sums, np.float64(top_p[r]) * sums[-1]) + 1]
            kept = kept[: max(1, np.count_nonzero(kept >= np.float64(min_p[r])))]
            sums = np.cumsum(kept)
            at = min(np.searchsorted(sums, u[r] * sums[-1], side="right"), len(kept) - 1)
            tokens[r], logprobs[r] = order[at], np.log(kept[at]) - np.log(sums[-1])
        return tokens, logprobs
    pool, q, lens, tables = _shared_inputs(case, seed)
    rows, hkv = case["rows"], case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    x = q.double().view(len(lens), rows, hkv, case["heads"] // hkv, -1)
    for i, (n, table) in enumerate(zip(lens, tables)):
        blocks = pool[:, torch.from_numpy(table.astype(np.int64)).cuda()].double()      # K and V [2, blocks, heads, BLOCK, features]
        for h in range(hkv):
            k, v = blocks[:, :, h].flatten(1, 2)
            for r in range(rows):
                a = (x[i, r, h] @ k[: n + r + 1].T) * case["head_dim"] ** -0.5
                if case["softcap"]:
                    a = torch.tanh(a / case["softcap"]) * case["softcap"]
                out.view_as(x)[i, r, h] = torch.softmax(a, -1) @ v[: n + r + 1]
    return out.reshape(q.shape[0], -1)
