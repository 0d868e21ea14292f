"""Attention of sequences that share a prefix: the bits of paged_attention for every row, whatever is shared by whom, and the
formula in 64 bits. Against that the 2-norm of the error is that of rounding the output to bf16 (half a step, 2^-9 of a value
at the most: 1.7e-3 of the norm on the average of mantissas) and of its fp32 parts, far below."""
import numpy as np
import pytest
import torch

from kiln_b200 import api
from kiln_b200.synth import PRESETS, synth_checkpoint

pytestmark = pytest.mark.gpu


def pools(ctx, kv_heads, dim, blocks, block_size, seed, layers=1, std=1.0):
    """Random K and V, written through rope_kv_write without a rotation: (PagedKv, [layers, 2, blocks, kv heads, block, dim])."""
    kv = api.PagedKv(ctx, api.KvSpec(layers, kv_heads, dim, blocks, block_size))
    g = torch.Generator(device="cuda").manual_seed(seed)
    data = torch.empty(layers, 2, blocks, kv_heads, block_size, dim, device="cuda").normal_(0, std, generator=g).to(torch.bfloat16)
    for layer in range(layers):
        k, v = (t.transpose(1, 2).reshape(-1, kv_heads * dim) for t in data[layer])
        seq = api.SeqStep(blocks * block_size, 0, 0, np.arange(blocks, dtype=np.uint32))
        api.rope_kv_write(ctx, kv, layer, torch.cat([k, k, v], 1), torch.zeros(dim // 2, device="cuda"), kv_heads, [seq])
    return kv, data


def tables(groups, block_size, seed):
    """groups: [(shared tokens, [(len, offset), ..]), ..] -> SeqSteps over permuted blocks, and the number of blocks. The first
    shared // block_size blocks of a group's tables are the same."""
    want = []
    for shared, members in groups:
        first = shared // block_size
        want.append((first, [(ln, off, -(-(ln + off) // block_size)) for ln, off in members]))
    total = sum(f + sum(n - f for _, _, n in m) for f, m in want)
    order, at, seqs = np.random.default_rng(seed).permutation(total), 0, []
    for first, members in want:
        head = order[at: at + first]
        at += first
        for ln, off, n in members:
            seqs.append(api.SeqStep(ln, off, 0, np.concatenate([head, order[at: at + n - first]]).astype(np.uint32)))
            at += n - first
    return seqs, total


def formula(data, q, seqs, scale, softcap):
    hkv, dim, rows = data.shape[2], data.shape[4], []
    at = 0
    for s in seqs:
        k, v = (t[torch.from_numpy(s.blocks.astype(np.int64)).cuda()].transpose(1, 2).reshape(-1, hkv, dim).double() for t in data)
        for r in range(s.len):
            n = s.offset + r + 1
            x = q[at].double().view(hkv, -1, dim)
            a = torch.einsum("hgd,khd->hgk", x, k[:n]) * scale
            if softcap:
                a = softcap * torch.tanh(a / softcap)
            rows.append(torch.einsum("hgk,khd->hgd", torch.softmax(a, -1), v[:n]).reshape(-1))
            at += 1
    return torch.stack(rows)


def close(out, want):
    assert float((out.double() - want).norm() / want.norm()) < 2.0e-3
    assert float((out.double() - want).abs().max()) <= 2 ** -8 * float(want.abs().max())


def run_both(ctx, kv, data, heads, seqs, seed, softcap=0.0, scale=None, layer=0, std=1.5):
    n, dim = sum(s.len for s in seqs), data.shape[-1]
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.empty(n, heads, dim, device="cuda").normal_(0, std, generator=g).to(torch.bfloat16)
    scale = dim ** -0.5 if scale is None else scale
    plan = api.AttentionPlan(ctx, kv, heads, seqs)
    got = plan.run(layer, q, scale, softcap)
    torch.cuda.synchronize()
    want = api.paged_attention(ctx, kv, layer, q, seqs, scale, softcap)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    return q, got, plan


HEADS = [(32, 8, 128), (28, 4, 128), (32, 8, 64), (16, 8, 256), (8, 8, 128), (24, 1, 64), (64, 1, 128)]
SHARED = {   # what 30 to 150 sequences share; enough for it to be read once with a kv head alone too
    "whole chunks": [(2048, [(1, 2048 + i) for i in range(80)])],
    "ends on its edge": [(1536, [(1, 1535 + i % 3) for i in range(150)])],          # the ones whose own row stands in the last chunk don't share it
    "not a block's multiple": [(2001, [(1, 2001 + 29 * i) for i in range(90)])],
    "verify rows": [(1600, [(5, 1700 + i) for i in range(70)])],
    "ragged rows": [(2560, [(1 + i % 6, 2600 + 61 * i) for i in range(60)])],
    "two groups and loners": [(0, [(1, 700)]), (2048, [(1, 2100 + i) for i in range(60)]), (0, [(1, 3), (1, 0), (2, 1500)]), (3000, [(1 + i % 2, 3050 + 40 * i) for i in range(50)])],
    "few": [(8192, [(1, 8200 + i) for i in range(30)])],
}


def shares(plan):
    read, apart = plan.keys()
    return read < apart


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("name", list(SHARED))
def test_rows_have_the_bits_that_they_have_alone(ctx, heads, kv_heads, dim, name):
    seqs, total = tables(SHARED[name], 16, len(name))
    kv, data = pools(ctx, kv_heads, dim, total, 16, 5)
    softcap = 30.0 if dim == 256 else 0.0
    q, got, plan = run_both(ctx, kv, data, heads, seqs, 7, softcap)
    # with 24 heads to a kv head and more, several rows of one sequence fill a unit by themselves
    assert shares(plan) or (heads // kv_heads >= 24 and any(s.len > 1 for s in seqs))
    close(got, formula(data[0], q, seqs, dim ** -0.5, softcap))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("groups", [
    [(512, [(1, 512), (1, 600)])], [(0, [(1, 900), (1, 800)])], [(496, [(1, 900 + i) for i in range(200)])], [(2000, [(4, 2040)])], [(0, [(1, 0)])],
    [(1024, [(130, 1024)] + [(1, 1200 + i) for i in range(90)])]])
def test_what_is_not_shared(ctx, groups):
    """Too little to be read once, less than a chunk, one sequence, no history, beside a piece of a prompt."""
    seqs, total = tables(groups, 16, 1)
    kv, data = pools(ctx, 4, 128, total, 16, 5)
    q, got, plan = run_both(ctx, kv, data, 16, seqs, 7)
    assert not shares(plan)
    close(got, formula(data[0], q, seqs, 128 ** -0.5, 0.0))


@pytest.mark.parametrize("block_size", [16, 32, 64, 128])
@pytest.mark.parametrize("softcap,scale", [(0.0, None), (20.0, None), (0.0, -0.1), (0.0, 0.0), (5.0, 3.0)])
def test_block_sizes_caps_and_scales(ctx, block_size, softcap, scale):
    seqs, total = tables([(2048, [(2, 2100 + 11 * i) for i in range(50)])], block_size, 3)
    kv, data = pools(ctx, 2, 128, total, block_size, 9)
    _, _, plan = run_both(ctx, kv, data, 8, seqs, 1, softcap, scale)
    assert shares(plan)


def test_a_tree_of_prefixes(ctx):
    """All share two chunks, eights of them two more, and some in the middle another one: every chunk goes by who has it in common."""
    bs, rng = 16, np.random.default_rng(2)
    order = np.random.default_rng(2).permutation(4000)
    trunk, branches, deeper, at, seqs = order[:64], [order[64 * (1 + i): 64 * (2 + i)] for i in range(8)], order[640:672], 700, []
    for i in range(64):
        deep = 20 <= i < 40
        head = np.concatenate([trunk, branches[i // 8]] + ([deeper] if deep else []))
        off = len(head) * bs + int(rng.integers(0, 300))
        n = -(-(off + 1 + i % 3) // bs)
        own = order[at: at + n - len(head)]
        at += len(own)
        seqs.append(api.SeqStep(1 + i % 3, off, 0, np.concatenate([head, own]).astype(np.uint32)))
    kv, data = pools(ctx, 4, 128, 4000, bs, 4)
    q, got, plan = run_both(ctx, kv, data, 16, seqs, 3)
    # 64 tables share 1024 keys, read by units of 32 of their 127 tokens; eights 1024 more; 20 in the middle 512 in three runs, which
    # their branches' edges cut
    read, apart = plan.keys()
    assert apart - read == 1024 * (64 - 4) + 1024 * (64 - 8) + 512 * (20 - 3)
    close(got, formula(data[0], q, seqs, 128 ** -0.5, 0.0))


@pytest.mark.parametrize("early", [False, True])
def test_one_table_for_all(ctx, early):
    """Every block is shared, the rows' own among them, at different positions. Where one of them is written in a shared chunk nothing behind
    it is read for all."""
    kv, data = pools(ctx, 2, 128, 160, 16, 4)
    table = np.random.default_rng(0).permutation(160).astype(np.uint32)
    seqs = [api.SeqStep(3, 2000 + 8 * i, 0, table) for i in range(65)]
    if early:
        seqs += [api.SeqStep(3, off, 0, table) for off in (40, 600)]
    q, got, plan = run_both(ctx, kv, data, 8, seqs, 3)
    assert shares(plan) != early
    close(got, formula(data[0], q, seqs, 128 ** -0.5, 0.0))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (28, 4, 128), (32, 8, 64), (16, 8, 256), (64, 8, 128)])
@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("prefix", [512 + 300, 1024 + 511, 2048 + 130, 2048 + 400, 4096 + 511])
def test_a_prefix_that_ends_inside_a_chunk(ctx, heads, kv_heads, dim, rows, prefix):
    """The pieces of 128 keys that all have of the chunk are taken once, and every sequence goes on from there: in the middle of
    a maximum's life, of a sum and of an output. In two groups, one of single rows."""
    tails = np.random.default_rng(prefix).integers(1, 130, 390)
    tails[:4] = 1, 128, 512, 1100
    seqs, total = tables([(prefix // 16 * 16, [(rows, prefix + int(t)) for t in tails[:250]]), (prefix // 16 * 16, [(1, prefix + int(t)) for t in tails[250:]])], 16, 1)
    kv, data = pools(ctx, kv_heads, dim, total, 16, 4)
    for softcap in (0.0, 30.0):
        q, got, plan = run_both(ctx, kv, data, heads, seqs, 3, softcap)
        read, apart = plan.keys()
        pieces, per = prefix // 16 * 16 // 128, 128 // (heads // kv_heads)
        assert apart - read == pieces * 128 * (390 - -(-250 * rows // per) - -(-140 // per))
        close(got[: 5 * rows], formula(data[0], q[: 5 * rows], seqs[:5], dim ** -0.5, softcap))
    assert ctx.device_status() == 0


def test_scores_that_grow_behind_a_shared_piece(ctx):
    """The maximum of what is shared is outweighed by far behind it, and the other way round: what was summed before is scaled down, or
    what follows."""
    seqs, total = tables([(2048 + 256, [(1, 2048 + 256 + i) for i in range(160)])], 16, 1)
    own = sorted({int(b) for s in seqs for b in s.blocks[(2048 + 256) // 16:]})
    for loud, std in ((1.0, 0.05), (1.0, 40.0), (30.0, 1.0), (1 / 30, 1.0)):
        kv, data = pools(ctx, 8, 128, total, 16, 4, std=std)
        data[0, 0, own] *= loud            # their own keys
        k, v = (t.transpose(1, 2).reshape(-1, 8 * 128) for t in data[0])
        api.rope_kv_write(ctx, kv, 0, torch.cat([k, k, v], 1), torch.zeros(64, device="cuda"), 8, [api.SeqStep(total * 16, 0, 0, np.arange(total, dtype=np.uint32))])
        q, got, plan = run_both(ctx, kv, data, 32, seqs, 3, std=1.5)
        read, apart = plan.keys()
        assert apart - read == (2048 + 256) * (160 - 5)
        close(got, formula(data[0], q, seqs, 128 ** -0.5, 0.0))


def test_windows_layers_streams_and_graphs(ctx):
    """A plan serves all layers, windowed ones too, on whatever stream is the current one, and in a graph that is replayed after
    the queries and the pools have changed."""
    seqs, total = tables([(2048, [(2, 2060 + 20 * i) for i in range(50)])], 16, 1)
    kv, data = pools(ctx, 2, 128, total, 16, 4, layers=2)
    q, got, plan = run_both(ctx, kv, data, 8, seqs, 3, layer=1)
    assert shares(plan)
    scale = 128 ** -0.5
    for window in (1, 100, 600, 5000):
        w = plan.run(0, q, scale, 0.0, window)
        torch.cuda.synchronize()
        assert torch.equal(w, api.paged_attention(ctx, kv, 0, q, seqs, scale, 0.0, window))
    for stream in (torch.cuda.Stream(), torch.cuda.ExternalStream(ctx.stream)):
        with torch.cuda.stream(stream):
            x = torch.zeros_like(q)
            for _ in range(10):
                x.copy_(q)
                a = plan.run(1, x, scale)
                x.zero_()
        torch.cuda.synchronize()
        assert torch.equal(a, got)
    still, out = q.clone(), torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(0, still, scale, out=out)
        plan.run(1, still, scale, 10.0)
    ctx.sync()
    for turn in range(2):
        still.copy_(q if turn else -q)
        kv.copy_block(int(seqs[0].blocks[turn]), int(seqs[0].blocks[3]))
        ctx.sync()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, api.paged_attention(ctx, kv, 0, still, seqs, scale))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (16, 8, 256)])
def test_a_plan_is_set_step_after_step(ctx, heads, kv_heads, dim):
    """One plan for steps that follow one another without a wait: more rows and fewer, with what is shared and without, capped
    (which may want other units) and not. Every step has paged_attention's bits. A graph ends the setting."""
    seqs, total = tables([(2048, [(4, 2100 + 20 * i) for i in range(50)]), (0, [(1, 300), (40, 0)])], 16, 1)
    kv, _ = pools(ctx, kv_heads, dim, total, 16, 4)
    steps = [[api.SeqStep(n, s.offset + at, 0, s.blocks) for s in seqs[:50]] for at, n in ((0, 1), (1, 1), (2, 2))]
    steps += [seqs[50:], seqs, seqs[3:4], steps[0]]
    q = torch.randn(sum(s.len for s in seqs), heads, dim, device="cuda").to(torch.bfloat16)
    plan, got, sharing = api.AttentionPlan(ctx, kv, heads, seqs[50:51]), [], []
    torch.cuda.synchronize()
    for step in steps:
        plan.set(step)
        assert plan.tokens == sum(s.len for s in step)
        sharing.append(shares(plan))
        got.append([plan.run(0, q[: plan.tokens], dim ** -0.5, cap) for cap in (0.0, 20.0)])
    with pytest.raises(api.KcError):
        plan.set([api.SeqStep(1, -1, 0, seqs[0].blocks)])
    assert plan.tokens == 50
    got.append([plan.run(0, q[:50], dim ** -0.5, cap) for cap in (0.0, 20.0)])
    torch.cuda.synchronize()
    assert sharing == [True, True, True, False, False, False, True]     # a step with 40 rows of a prompt keeps to the sequences' own units
    for step, outs in zip(steps + steps[:1], got):
        n = sum(s.len for s in step)
        for out, cap in zip(outs, (0.0, 20.0)):
            assert torch.equal(out, api.paged_attention(ctx, kv, 0, q[:n], step, dim ** -0.5, cap))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plan.run(0, q[:50], dim ** -0.5)
    with pytest.raises(api.KcError):
        plan.set(steps[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, got[0][0])


def test_large_scores(ctx):
    """One key outweighs all others by far: maxima that move by thousands of binary orders from chunk to chunk."""
    seqs, total = tables([(2048, [(1, 2060 + 9 * i) for i in range(80)])], 16, 1)
    kv, data = pools(ctx, 2, 64, total, 16, 4, std=40.0)
    q, got, plan = run_both(ctx, kv, data, 8, seqs, 3, std=40.0)
    assert shares(plan)
    close(got, formula(data[0], q, seqs, 64 ** -0.5, 0.0))


def test_rows_past_the_shared_ones_are_left(ctx):
    seqs, total = tables([(2048, [(1, 2048)] * 90)], 16, 1)
    kv, data = pools(ctx, 2, 64, total, 16, 4)
    q = torch.randn(90, 8, 64, device="cuda").to(torch.bfloat16)
    out = torch.full((92, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    plan = api.AttentionPlan(ctx, kv, 8, seqs)
    assert shares(plan)
    plan.run(0, q, 0.125, out=out[1:91])
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[91] == 7).all() and torch.equal(out[1:91], api.paged_attention(ctx, kv, 0, q, seqs, 0.125))


@pytest.mark.parametrize("n,rows,shared", [(100, 3, 1040), (500, 1, 1408)])     # the second one behind pieces of a chunk too
def test_a_models_steps_share(ctx, n, rows, shared):
    """A model's verify step over sequences that share a prompt: the logits of a sequence are those it has alone, bit for bit, and
    the K/V it writes too; sampled tokens and counts follow."""
    cfg = PRESETS["tiny-llama-d128"]
    model = api.CudaModel(ctx, cfg, synth_checkpoint(cfg, seed=1), max_step_tokens=512, max_step_seqs=512)
    rng, first = np.random.default_rng(1), shared // 16
    kv = api.PagedKv(ctx, model.kv_spec(first + 4 * n + 4, 16))
    prompt = rng.integers(0, cfg.vocab_size, shared).tolist()
    for at in range(0, shared, 512):
        piece = prompt[at: at + 512]
        model.forward_step(api.StepBatch(piece, [api.SeqStep(len(piece), at, 0, np.arange(first, dtype=np.uint32))]), kv)
    own = [np.arange(first + 4 * i, first + 4 + 4 * i, dtype=np.uint32) for i in range(n)]
    ids = rng.integers(0, cfg.vocab_size, (n, rows))
    seqs = [api.SeqStep(rows, shared, rows, np.concatenate([np.arange(first, dtype=np.uint32), own[i]])) for i in range(n)]
    plan = api.AttentionPlan(ctx, kv, cfg.num_attention_heads, seqs)
    read, apart = plan.keys()
    assert apart - read >= shared // 128 * 128 * n * 0.8
    batch = api.StepBatch(ids.reshape(-1).tolist(), seqs)
    logits = model.forward_step(batch, kv)
    ctx.sync()
    together = logits.clone()
    wrote = kv.read_block_bytes(int(own[7][0]))
    for i in (0, 7, 50, n - 1):
        kv.copy_block(first + 4 * n, int(own[i][0]))      # what it wrote is written again
        alone = model.forward_step(api.StepBatch(ids[i].tolist(), [seqs[i]]), kv)
        ctx.sync()
        assert torch.equal(alone.view(torch.int16), together[rows * i: rows * (i + 1)].view(torch.int16))
    assert kv.read_block_bytes(int(own[7][0])) == wrote
    committed, ncom, nacc = model.verify_step(batch, kv)
    assert torch.equal(torch.from_numpy(committed.astype(np.int64)).cuda(), api.greedy_rows(ctx, together).long())
    assert ctx.device_status() == 0


def test_refusals(ctx):
    live = api.live_objects()
    kv, _ = pools(ctx, 2, 64, 40, 16, 4)
    good = [api.SeqStep(1, 20, 0, np.arange(4, dtype=np.uint32))]
    for heads, seqs in ((3, good), (0, good), (2 * 65, good), (8, []), (8, [api.SeqStep(0, 3, 0, good[0].blocks)]), (8, [api.SeqStep(1, -1, 0, good[0].blocks)]),
                        (8, [api.SeqStep(1, 64, 0, good[0].blocks)]), (8, [api.SeqStep(1, 3, 0, np.array([40], dtype=np.uint32))])):
        with pytest.raises(api.KcError):
            api.AttentionPlan(ctx, kv, heads, seqs)
    plan = api.AttentionPlan(ctx, kv, 8, good)
    q = torch.zeros(1, 8, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (q.float(), q[:, :4], q.expand(2, 8, 64), q.cpu(), torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")[:, :, ::2]):
        with pytest.raises(ValueError):
            plan.run(0, bad, 1.0)
    for layer in (-1, 1):
        with pytest.raises(api.KcError):
            plan.run(layer, q, 1.0)
    with pytest.raises(api.KcError):
        plan.run(0, torch.zeros(513, dtype=torch.bfloat16, device="cuda")[1:].view(1, 8, 64), 1.0)
    plan.run(0, q, 1.0)
    ctx.sync()
    kv.close()
    for call in (lambda: plan.run(0, q, 1.0), lambda: plan.set(good)):
        with pytest.raises(ValueError):
            call()
    plan.close()
    for call in (lambda: plan.run(0, q, 1.0), lambda: plan.set(good)):
        with pytest.raises(ValueError):
            call()
    assert api.live_objects() == live
