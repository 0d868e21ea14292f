"""Drawn rows against the definition in 64 bits, at the sizes, masks, values and settings where they can go wrong; and the verify
round whose rows are drawn. Tokens have to be equal. The log probability is rounded once from 64 bits: half a step of fp32 of its
value, and what a logarithm near 1 loses of a share that is itself 1e-13 off.
"""
import math

import numpy as np
import pytest
import torch

from kiln_b200 import api
from kiln_b200.synth import PRESETS, synth_checkpoint
from oracle.bookkeeping import settle_walk

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24     # half a step of fp32, relative


def draw_row(row, temperature, top_k, top_p, min_p, u):
    """(token, log probability) of one row by the definition."""
    row = np.asarray(row, dtype=np.float64) + 0.0
    row = np.where(np.isnan(row), -np.inf, row)
    order = np.argsort(-row, kind="stable")
    order = order[row[order] > -np.inf]
    if not len(order):
        return 0, -np.inf
    if not temperature > 0:
        return int(order[0]), 0.0
    top = row[order[0]]
    with np.errstate(all="ignore"):
        far = np.where(row[order] == top, 0.0, row[order] - top)
        w = np.where(far == 0, 1.0, np.where(far == -np.inf, 0.0, np.exp(far / np.float64(temperature))))   # beside an infinite logit
    kept = w[:top_k] if top_k > 0 else w
    if top_p < 1:
        sums = np.cumsum(kept)
        kept = kept[: np.searchsorted(sums, np.float64(top_p) * sums[-1]) + 1]
    if min_p > 0:
        kept = kept[: max(1, np.count_nonzero(w >= np.float64(min_p)))]
    sums = np.cumsum(kept)
    at = len(kept) - 1 if not u < 1 else min(int(np.searchsorted(sums, np.float64(u) * sums[-1], side="right")), len(kept) - 1)
    return int(order[at]), float(np.log(kept[at] / sums[-1]))


def raw_settings(settings):
    """Settings as they are, also the ones that SamplingParams refuses."""
    return torch.from_numpy(np.array(settings, dtype=[("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")]).view(np.int32).reshape(-1, 4)).cuda()


def check(ctx, logits, settings, u):
    """logits: a bf16 CUDA tensor [rows, vocab]."""
    u = torch.tensor(u, dtype=torch.float32, device="cuda")
    tokens, logprobs = api.sample_rows(ctx, logits, raw_settings(settings), u)
    torch.cuda.synchronize()
    host = logits.float().cpu().numpy()
    for r, (s, x) in enumerate(zip(settings, u.tolist())):
        s = (np.float32(s[0]), s[1], np.float32(s[2]), np.float32(s[3]))
        token, logprob = draw_row(host[r], *s, x)
        assert int(tokens[r]) == token, (r, s, x)
        got = float(logprobs[r])
        assert got == logprob or abs(got - logprob) <= STEP * abs(logprob) + 1e-12, (r, s, x, got, logprob)


def language(rows, vocab, seed, std=2.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.empty(rows, vocab).normal_(0, std, generator=g)
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 9.0
    return x.to(torch.bfloat16).cuda()


def mixed(rows, rng):
    return [(float(rng.choice([0.3, 0.7, 1.0, 1.0, 1.5, 0.0])), int(rng.choice([0, 0, 1, 5, 40, 1000])), float(rng.choice([1.0, 1.0, 0.1, 0.9, 0.95])),
             float(rng.choice([0.0, 0.0, 0.02, 0.3]))) for _ in range(rows)]


@pytest.mark.parametrize("rows", [1, 3, 40, 90, 170, 310])      # 8, 4, 2 and 1 CTAs a row
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 257, 4099, 50001])
def test_rows_are_drawn_by_the_definition(ctx, rows, vocab):
    rng = np.random.default_rng(rows * 100003 + vocab)
    check(ctx, language(rows, vocab, rows + vocab), mixed(rows, rng), rng.random(rows).astype(np.float32).clip(0, 1 - 2 ** -24).tolist())


@pytest.mark.parametrize("vocab", [128256, 152064, 256000])
def test_whole_vocabularies(ctx, vocab):
    rng = np.random.default_rng(vocab)
    check(ctx, language(12, vocab, vocab), mixed(12, rng), rng.random(12).astype(np.float32).clip(0, 1 - 2 ** -24).tolist())


ODD = {
    "equal": lambda g, n: torch.full((n,), 1.5),
    "zeros of either sign": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.5, 0.0, -0.0),
    "zeros and others": lambda g, n: torch.randint(-1, 2, (n,), generator=g).float(),
    "all magnitudes": lambda g, n: torch.randn(n, generator=g).sign() * torch.exp2(torch.empty(n).uniform_(-133, 127, generator=g)),
    "tiny": lambda g, n: torch.randn(n, generator=g) * 2.0 ** -40,
    "subnormal": lambda g, n: torch.randn(n, generator=g) * 2.0 ** -130,
    "huge": lambda g, n: torch.randn(n, generator=g) * 2.0 ** 100,
    "negative": lambda g, n: -100 - 50 * torch.rand(n, generator=g),
    "one of few": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.99, -math.inf, torch.randn(n, generator=g)),
    "masked": lambda g, n: torch.full((n,), -math.inf),
    "masked but the last": lambda g, n: torch.cat([torch.full((n - 1,), -math.inf), torch.tensor([-3.0])]),
    "lowest value": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.9, torch.finfo(torch.bfloat16).min, torch.randn(n, generator=g)),
    "nan": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.3, math.nan, torch.randn(n, generator=g)),
    "all nan": lambda g, n: torch.full((n,), math.nan),
    "infinite": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.1, math.inf, torch.randn(n, generator=g)),
    "both infinities": lambda g, n: torch.tensor([math.inf, -math.inf]).repeat(n)[:n],
}
EDGES = [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0), (1e-45, 3, 0.5, 0.5), (1e30, 0, 1.0, 0.0), (math.inf, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0),
         (0.8, 7, 0.9, 0.0), (0.8, 0, 1e-9, 0.0), (0.8, 0, 0.0, 0.0), (0.8, 0, -1.0, 0.0), (0.8, 0, 2.0, 0.0), (1.3, 0, 1.0, 1.0), (1.3, 0, 0.7, 1e-6), (1.3, 1 << 30, 0.999999, 0.0),
         (1.3, -5, 1.0, -1.0), (-1.0, 5, 0.5, 0.5), (math.nan, 5, 0.5, 0.5)]
NUMBERS = [0.0, 2.0 ** -30, 0.25, 0.5, 0.73, 1 - 2.0 ** -24]


@pytest.mark.parametrize("values", list(ODD))
@pytest.mark.parametrize("vocab", [5, 1003])
def test_odd_rows_and_settings(ctx, values, vocab):
    g = torch.Generator().manual_seed(len(values) * 7 + vocab)
    settings = [s for s in EDGES for _ in NUMBERS]
    rows = torch.stack([ODD[values](g, vocab) for _ in settings]).to(torch.bfloat16).cuda()
    check(ctx, rows, settings, NUMBERS * len(EDGES))
    check(ctx, rows[:6].contiguous(), settings[:6], NUMBERS)     # the same with eight CTAs a row


def test_many_equal_values(ctx):
    """More of one value than 16 bits count, and the occurrence that is drawn lies anywhere among them."""
    n = 200003
    row = torch.full((9, n), 0.25, dtype=torch.bfloat16, device="cuda")
    row[:, 77] = 3.0
    row[3:6, ::2] = -0.5
    u = [0.0, 0.3, 1 - 2.0 ** -24] * 3
    check(ctx, row, [(1.0, 0, 1.0, 0.0)] * 6 + [(1.0, 100000, 0.9, 0.0), (2.0, 0, 0.4, 0.01), (1.0, 0, 1.0, 0.05)], u)


def test_numbers_outside_their_range(ctx):
    x = language(4, 999, 5)
    u = torch.tensor([-0.5, 1.0, 7.0, math.nan], device="cuda")
    tokens, _ = api.sample_rows(ctx, x, [api.SamplingParams(1.0, 20)] * 4, u)
    host = x.float().cpu().numpy()
    for r in range(4):
        order = np.argsort(-host[r].astype(np.float64), kind="stable")
        assert int(tokens[r]) == order[0 if r == 0 else 19]


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("ld", [1009, 1016])
def test_strides_and_alignment(ctx, shift, ld):
    """Rows of a wider tensor that start anywhere; what lies around them is larger than they are."""
    rng = np.random.default_rng(shift)
    wide = torch.full((11, ld), 50.0, dtype=torch.bfloat16, device="cuda")
    x = wide[:, shift: shift + 1000]
    x.copy_(language(11, 1000, shift))
    check(ctx, x, mixed(11, rng), rng.random(11).astype(np.float32).tolist())


def test_rows_do_not_hang_on_their_number(ctx):
    """A row has the same token and the same bits of its log probability with 8, 4, 2 and 1 CTAs."""
    rng = np.random.default_rng(3)
    x, settings, u = language(300, 30011, 11), raw_settings(mixed(300, rng)), torch.tensor(rng.random(300).astype(np.float32), device="cuda")
    want, p = api.sample_rows(ctx, x, settings, u)
    for n in (1, 20, 50, 100):
        got, q = api.sample_rows(ctx, x[:n], settings[:n], u[:n])
        assert torch.equal(got, want[:n]) and torch.equal(q.view(torch.int32), p[:n].view(torch.int32))


@pytest.mark.parametrize("rows", [1, 40, 80, 200])
@pytest.mark.parametrize("vocab", [9, 300, 5003, 128256])
def test_values_below_all_others(ctx, rows, vocab):
    """One value of a magnitude far below the rest's, of either sign or both, a zero or NaN as it may be, or two: in the middle of a row,
    at its end, as its largest."""
    rng = np.random.default_rng(rows + vocab)
    tiny = [2.0 ** -26, -2.0 ** -26, 1e-30, -1e-30, 0.0, -0.0, math.nan, 1e-40, -1e-40, 2.0 ** -25 * 0.99]
    x = language(rows, vocab, 17)
    host = x.float().cpu()
    host[::3] = -host[::3].abs() - 0.5                   # below zero: a tiny value is the largest
    for r in range(rows):
        places = rng.choice(vocab, 3, replace=False)
        if r % 4 == 3:
            places[0] = vocab - 1
        for k in range([1, 1, 2, 1, 3][r % 5]):
            host[r, places[k]] = tiny[(r // 2 + 3 * k) % len(tiny)]
    settings = [(float(rng.choice([0.7, 1.0, 100.0])), int(rng.choice([0, 1, 2, 40])), float(rng.choice([1.0, 0.5, 0.95])), float(rng.choice([0.0, 0.3, 1.0]))) for _ in range(rows)]
    check(ctx, host.to(torch.bfloat16).cuda(), settings, rng.choice([0.0, 0.3, 0.999, 1 - 2 ** -24], rows).astype(np.float32).tolist())


@pytest.mark.parametrize("rows,vocab", [(160, 270001), (80, 530003), (1, 1048569), (1, 1200000)])
def test_long_rows(ctx, rows, vocab):
    """More values than a bin has room to say where they stand (8 to the vector, 16384 vectors a CTA), and just as many."""
    rng = np.random.default_rng(vocab)
    check(ctx, language(rows, vocab, 3)[: rows], mixed(rows, rng), rng.random(rows).astype(np.float32).clip(0, 1 - 2 ** -24).tolist())


@pytest.mark.parametrize("rows,vocab", [(310, 50001), (310, 4099), (90, 4099), (40, 257), (1, 8)])
def test_every_run_counts_every_token(ctx, rows, vocab):
    """The same rows many times over: a token that one run did not count would show in the log probability."""
    logits = language(rows, vocab, 5)
    params = api.pack_sampling([api.SamplingParams()] * rows, logits.device)
    u = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    first = [t.clone() for t in api.sample_rows(ctx, logits, params, u)]
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        tokens, logprobs = api.sample_rows(ctx, logits, params, u)
        wrong += (tokens != first[0]).sum() + (logprobs != first[1]).sum()
    assert int(wrong) == 0
    check(ctx, logits[:5], [(1.0, 0, 1.0, 0.0)] * min(rows, 5), u[:5].tolist())


def test_streams_and_graphs(ctx):
    """Part of whatever stream is torch's current one, of the context's own, and of a graph that is replayed with new rows."""
    x, u = language(5, 4099, 1), torch.tensor([0.1, 0.4, 0.6, 0.8, 0.95], device="cuda")
    params = api.pack_sampling([api.SamplingParams(0.9, 0, 0.97, 0.0)] * 5, "cuda")
    other = language(5, 4099, 2)
    want, want_other = (api.sample_rows(ctx, v, params, u)[0].clone() for v in (x, other))
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.ExternalStream(ctx.stream)):
        with torch.cuda.stream(stream):
            y = torch.empty_like(x)
            for _ in range(20):
                y.copy_(other)
                a = api.sample_rows(ctx, y, params, u)[0]
                y.copy_(x)
                b = api.sample_rows(ctx, y, params, u)[0]
        torch.cuda.synchronize()
        assert torch.equal(a, want_other) and torch.equal(b, want)
    still, out, lp = x.clone(), torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.sample_rows(ctx, still, params, u, out=out, logprobs=lp)
    for source, expected in ((other, want_other), (x, want)):
        still.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected)
    api.sample_rows(ctx, x, params, u)                             # and outside again
    ctx.sync()


def test_refusals(ctx):
    x, u, params = language(3, 100, 1), torch.zeros(3, device="cuda"), api.pack_sampling([api.SamplingParams()] * 3, "cuda")
    for bad in (dict(logits=x.float()), dict(logits=x.t()), dict(logits=x[0]), dict(uniforms=u.double()), dict(uniforms=u[:2]), dict(params=params[:2]),
                dict(params=params.cpu()), dict(uniforms=u.cpu()), dict(out=torch.zeros(3, dtype=torch.int64, device="cuda")),
                dict(logprobs=torch.zeros(6, device="cuda")[::2]), dict(params=[api.SamplingParams()] * 2)):
        with pytest.raises(ValueError):
            api.sample_rows(ctx, **{**dict(logits=x, params=params, uniforms=u), **bad})
    with pytest.raises(api.KcError):                               # rows that lie in one another
        api.sample_rows(ctx, x[:1].expand(3, 100), params, u)
    assert api.sample_rows(ctx, x, params, u)[0].shape == (3,)


# ---- the verify round with drawn rows -----------------------------------------------------------------------------

@pytest.fixture(scope="module")
def small(ctx):
    cfg = PRESETS["tiny-llama"]
    return cfg, api.CudaModel(ctx, cfg, synth_checkpoint(cfg, seed=3), max_step_tokens=64, max_step_seqs=8)


def prompts(model, ctx, n, length, vocab, same=False):
    rng = np.random.default_rng(5)
    kv = api.PagedKv(ctx, model.kv_spec(8 * n, 16))
    tables = [list(range(8 * i, 8 * i + 8)) for i in range(n)]
    ids = rng.integers(0, vocab, length).tolist()
    for t in tables:
        model.verify_step(api.StepBatch(ids if same else rng.integers(0, vocab, length).tolist(), [api.SeqStep(length, 0, 0, t)]), kv)
    return kv, tables, rng


def test_verify_round_draws_its_rows(ctx, small):
    """Row tokens are those of sample_rows over the forward's logits, counts those of the walk; rows without temperature are the
    greedy round's; a sequence that samples nothing gets nothing."""
    cfg, model = small
    kv, tables, rng = prompts(model, ctx, 5, 40, cfg.vocab_size)
    rows = [4, 1, 3, 4, 0]
    lens = [4, 1, 3, 4, 2]
    ids = rng.integers(0, cfg.vocab_size, sum(lens)).tolist()
    batch = api.StepBatch(ids, [api.SeqStep(n, 40, r, t) for n, r, t in zip(lens, rows, tables)])
    settings = [api.SamplingParams(0.8, 50, 0.95, 0.0), api.SamplingParams(1.2), api.SamplingParams(0.0, 3, 0.5, 0.5), api.SamplingParams(1.0, 0, 1.0, 0.01),
                api.SamplingParams(1.0)]
    logits = model.forward_step(batch, kv)
    ctx.sync()
    logits = logits.clone()
    greedy = model.verify_step(batch, kv)[0]
    for trial in range(8):
        u = rng.random(sum(rows)).astype(np.float32).clip(0, 1 - 2 ** -24)
        want, lp = api.sample_rows(ctx, logits, [s for s, r in zip(settings, rows) for _ in range(r)], torch.from_numpy(u).cuda())
        want = want.cpu().numpy()
        want[5:8] = greedy[5:8]
        # drafts that the first two rows of sequence 0 draw, and of the greedy one
        at = 0
        drafts = []
        for i, r in enumerate(rows):
            d = ids[sum(lens[:i]) + 1: sum(lens[:i]) + r]
            drafts.append(d)
        got, ncom, nacc, glp = model.verify_step_sampled(batch, kv, settings, u)
        assert got.tolist() == want.tolist()
        lp = lp.cpu().numpy()
        lp[5:8] = 0
        assert glp.tolist() == lp.tolist()
        for i, r in enumerate(rows):
            com, acc = settle_walk(want[at: at + r].tolist(), drafts[i]) if r else ([], 0)
            assert (int(ncom[i]), int(nacc[i])) == (len(com), acc)
            at += r
    assert ctx.device_status() == 0


def test_a_draft_that_is_drawn_is_accepted(ctx, small):
    """Rows drawn one step at a time after a prompt, handed in as a draft after the same one with the same numbers: accepted, all of
    it, and the bits are the same."""
    cfg, model = small
    kv, tables, rng = prompts(model, ctx, 2, 33, cfg.vocab_size, same=True)
    s = [api.SamplingParams(0.9, 0, 0.9, 0.0)]
    u = rng.random(5).astype(np.float32)
    first = token = 7
    drawn = []
    for j in range(5):
        rows, _, _, lp = model.verify_step_sampled(api.StepBatch([token], [api.SeqStep(1, 33 + j, 1, tables[0])]), kv, s, u[j: j + 1])
        token = int(rows[0])
        drawn.append((token, float(lp[0])))
    draft = [t for t, _ in drawn[:4]]
    rows, ncom, nacc, lp = model.verify_step_sampled(api.StepBatch([first] + draft, [api.SeqStep(5, 33, 5, tables[1])]), kv, s, u)
    assert [int(t) for t in rows] == [t for t, _ in drawn]
    assert int(nacc[0]) == 4 and int(ncom[0]) == 5
    assert [float(p) for p in lp] == [p for _, p in drawn]


def test_all_greedy_is_the_verify_round(ctx, small):
    cfg, model = small
    kv, tables, rng = prompts(model, ctx, 3, 20, cfg.vocab_size)
    batch = api.StepBatch(rng.integers(0, cfg.vocab_size, 9).tolist(), [api.SeqStep(3, 20, 3, t) for t in tables])
    a = model.verify_step(batch, kv)
    b = model.verify_step_sampled(batch, kv, [api.SamplingParams(0.0)] * 3, [0.5] * 9)
    assert all(np.array_equal(x, y) for x, y in zip(a, b[:3])) and not b[3].any()


def test_verify_round_refuses_bad_settings(ctx, small):
    cfg, model = small
    kv, tables, rng = prompts(model, ctx, 1, 20, cfg.vocab_size)
    batch = api.StepBatch([1, 2], [api.SeqStep(2, 20, 2, tables[0])])

    class Raw:
        def __init__(self, *v):
            self.temperature, self.top_k, self.top_p, self.min_p = v
    for bad in ((-1.0, 0, 1.0, 0.0), (math.nan, 0, 1.0, 0.0), (math.inf, 0, 1.0, 0.0), (1.0, -1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.5, 0.0), (1.0, 0, math.nan, 0.0),
                (1.0, 0, 1.0, -0.1), (1.0, 0, 1.0, 1.1)):
        with pytest.raises(api.KcError):
            model.verify_step_sampled(batch, kv, [Raw(*bad)], [0.1, 0.2])
    for u in ([0.1, 1.0], [-0.1, 0.2], [math.nan, 0.2]):
        with pytest.raises(api.KcError):
            model.verify_step_sampled(batch, kv, [api.SamplingParams()], u)
    with pytest.raises(ValueError):
        model.verify_step_sampled(batch, kv, [api.SamplingParams()], [0.1])
    with pytest.raises(ValueError):
        model.verify_step_sampled(batch, kv, [], [0.1, 0.2])
    assert len(model.verify_step_sampled(batch, kv, [api.SamplingParams()], [0.1, 0.2])[0]) == 2
