"""What the entry points that are queued without waiting refuse, and what their handles ask of the CUDA runtime, against a
stand-in for it. Needs no GPU; each test is a process of its own."""
import subprocess

import pytest

from tests.test_host_calls import ROOT, fake, run  # noqa: F401  (a fixture)


@pytest.fixture(scope="module")
def graphs(fake, tmp_path_factory):  # noqa: F811
    so = tmp_path_factory.mktemp("fake") / "fake_cudart_graphs.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I/usr/local/cuda/include", "-o", str(so), str(ROOT / "tests" / "fake_cudart_graphs.cpp")], check=True)
    return f"{fake}:{so}"


PLAN = """
def steps(lens, n_blocks=None, blocks=table):
    return (L.KcSeqStep * max(1, len(lens)))(*[L.KcSeqStep(n, off, 0, -(-(n + off) // 16) if n_blocks is None else n_blocks, blocks) for n, off in lens])
def create(lens, heads=4, **kw):
    p = C.c_void_p()
    return lib.kc_attn_plan_create(ctx, kv, steps(lens, **kw), len(lens), heads, C.byref(p)), p
def launches():
    return [c for c in calls() if c.startswith("launch")]
"""


def test_plans_are_refused(graphs):
    run(graphs, PLAN + """
before = lib.kc_live_objects()
far = (C.c_uint32 * 80)(*range(1, 81))
for bad in (dict(lens=[]), dict(lens=[(0, 5)]), dict(lens=[(1, 5), (0, 5)]), dict(lens=[(-1, 5)]), dict(lens=[(1, -1)]), dict(lens=[(1, 5)], heads=3), dict(lens=[(1, 5)], heads=0),
            dict(lens=[(1, 5)], heads=130), dict(lens=[(1, 40)], n_blocks=2), dict(lens=[(1, 1272)], blocks=far), dict(lens=[(1, 5)], blocks=None), dict(lens=[((1 << 24) + 1, 0)])):
    rc, p = create(**bad)
    assert rc == L.KC_ERR_INVALID and not p.value and lib.kc_last_error(), bad
for a in ((None, kv, steps([(1, 5)])), (ctx, None, steps([(1, 5)])), (ctx, kv, None)):
    assert lib.kc_attn_plan_create(*a, 1, 4, C.byref(C.c_void_p())) == L.KC_ERR_INVALID
assert lib.kc_attn_plan_create(ctx, kv, steps([(1, 5)]), 1, 4, None) == L.KC_ERR_INVALID
fake.fake_capture(1)
assert create([(1, 5)])[0] == L.KC_ERR_INVALID     # its copies are not part of a graph
fake.fake_capture(0)
assert lib.kc_live_objects() == before
rc, p = create([(3, 40), (1, 0)])
ok(rc)
def attend(plan=p, layer=0, q=at, out=at + 4 * 4 * 64 * 2):
    return lib.kc_attn_plan_run(plan, layer, q, 0.125, 0.0, 0, out)
fake.fake_reset()
for bad in (dict(plan=None), dict(layer=-1), dict(layer=1), dict(q=None), dict(q=at + 8), dict(out=None), dict(out=at + 4 * 4 * 64 * 2 + 2), dict(out=at), dict(out=at + 4 * 4 * 64 * 2 - 16), dict(q=at + 16, out=at)):
    assert attend(**bad) == L.KC_ERR_INVALID, bad
assert lib.kc_attn_plan_keys(None, C.byref(C.c_int64()), C.byref(C.c_int64())) == L.KC_ERR_INVALID
assert lib.kc_attn_plan_set(None, steps([(1, 5)]), 1) == L.KC_ERR_INVALID and lib.kc_attn_plan_set(p, None, 1) == L.KC_ERR_INVALID
assert not launches()
ok(attend())
assert launches()
lib.kc_attn_plan_free(p)
lib.kc_attn_plan_free(None)
assert lib.kc_live_objects() == before
""")


def test_a_plan_is_set_again(graphs):
    """No allocation while the plan has room, one copy a setting, no wait of the host; a refused step leaves the plan as it was."""
    run(graphs, PLAN + """
rc, p = create([(3, 40), (1, 0)])
ok(rc)
read, apart = C.c_int64(), C.c_int64()
def keys():
    ok(lib.kc_attn_plan_keys(p, C.byref(read), C.byref(apart)))
    return apart.value
assert keys() == 43 + 1
fake.fake_reset()
for off in range(41, 50):
    ok(lib.kc_attn_plan_set(p, steps([(3, off)]), 1))
    assert keys() == off + 3
assert calls() == ["copy"] * 9
assert lib.kc_attn_plan_set(p, steps([(3, -1)]), 1) == L.KC_ERR_INVALID and lib.kc_attn_plan_set(p, steps([]), 0) == L.KC_ERR_INVALID
assert keys() == 52 and not calls()
q, out = at, at + (1 << 19)
ok(lib.kc_attn_plan_run(p, 0, q, 0.125, 0.0, 0, out))
fake.fake_fail_above(1 << 16)                      # a step that the plan has no room for, and no memory for it
assert lib.kc_attn_plan_set(p, steps([(1, 1200)] * 600), 600) == L.KC_ERR_OOM
assert lib.kc_attn_plan_run(p, 0, q, 0.125, 0.0, 0, out) == L.KC_ERR_INVALID
fake.fake_fail_above(2 ** 62)
ok(lib.kc_attn_plan_set(p, steps([(1, 1200)] * 60), 60))
ok(lib.kc_attn_plan_run(p, 0, q, 0.125, 0.0, 0, out))
fake.fake_capture(1)
assert lib.kc_attn_plan_set(p, steps([(1, 5)]), 1) == L.KC_ERR_INVALID
ok(lib.kc_attn_plan_run(p, 0, q, 0.125, 0.0, 0, out))
fake.fake_capture(0)
assert lib.kc_attn_plan_set(p, steps([(1, 5)]), 1) == L.KC_ERR_INVALID     # the graph needs the plan as it is
assert b"graph" in lib.kc_last_error()
ok(lib.kc_attn_plan_run(p, 0, q, 0.125, 0.0, 0, out))
lib.kc_attn_plan_free(p)
""")


def test_no_times_from_a_graph(graphs):
    """The profile's events have no time inside a graph: a capture while it is on is refused, behind it all is as ever."""
    run(graphs, PLAN + """
rc, p = create([(3, 40)])
ok(rc)
ok(lib.kc_profile_enable(ctx, 1))
def both():
    return {lib.kc_attn_plan_run(p, 0, at, 0.125, 0.0, 0, at + 4096), lib.kc_sample_rows(ctx, at, 100, 2, 100, at, at, at, None)}
assert both() == {L.KC_OK}
fake.fake_capture(1)
assert both() == {L.KC_ERR_INVALID}
ok(lib.kc_profile_enable(ctx, 0))
assert both() == {L.KC_OK}
""")


def test_adapters_are_refused(graphs):
    run(graphs, """
before = lib.kc_live_objects()
def create(n_in=64, n_out=48, slots=3, rank=20):
    p = C.c_void_p()
    return lib.kc_adapters_create(ctx, n_in, n_out, slots, rank, C.byref(p)), p
for bad in (dict(n_in=0), dict(n_in=-32), dict(n_in=48), dict(n_out=0), dict(slots=0), dict(slots=(1 << 20) + 1), dict(rank=0), dict(rank=-1)):
    assert create(**bad)[0] == L.KC_ERR_INVALID, bad
assert create(rank=129)[0] == L.KC_ERR_UNSUPPORTED
fake.fake_fail_above(1 << 12)
assert create()[0] == L.KC_ERR_OOM
fake.fake_fail_above(2 ** 62)
assert lib.kc_live_objects() == before
rc, bank = create()
ok(rc)
for a in ((-1, at, at, 4, 1.0), (3, at, at, 4, 1.0), (0, None, at, 4, 1.0), (0, at, None, 4, 1.0), (0, at, at, 21, 1.0), (0, at, at, -1, 1.0), (0, at, at, 4, float("nan")), (0, at, at, 4, float("inf"))):
    assert lib.kc_adapters_set(bank, *a, 0) == L.KC_ERR_INVALID, a
assert lib.kc_adapters_set(None, 0, at, at, 4, 1.0, 0) == L.KC_ERR_INVALID
ok(lib.kc_adapters_set(bank, 2, at, at, 20, 1.0, 0)); ok(lib.kc_adapters_set(bank, 2, None, None, 0, 0.0, 0))
def rows(*slots, m=None):
    p = C.c_void_p()
    return lib.kc_adapter_rows_create(ctx, (C.c_int32 * max(1, len(slots)))(*slots), len(slots) if m is None else m, C.byref(p)), p
for bad in (rows(), rows(0, m=-1), rows(0, m=(1 << 24) + 1), rows(0, -2)):
    assert bad[0] == L.KC_ERR_INVALID
rc, who = rows(2, -1, 0, 2)
ok(rc)
rc, past = rows(0, 3)
ok(rc)
out = at + (1 << 16)
def apply(bank=bank, who=who, x=at, y=out, out=out):
    return lib.kc_adapters_apply(bank, who, x, y, out)
fake.fake_reset()
x_bytes, y_bytes = 4 * 64 * 2, 4 * 48 * 2
for bad in (dict(bank=None), dict(who=None), dict(x=None), dict(y=None), dict(out=None), dict(who=past), dict(x=at + 2), dict(y=out + 1), dict(out=out + 1), dict(out=at), dict(out=at + x_bytes - 2),
            dict(x=at + 256, out=at + 256 - y_bytes + 2), dict(y=out + 2), dict(y=out + y_bytes - 2), dict(y=out - y_bytes + 2)):
    assert apply(**bad) == L.KC_ERR_INVALID, bad
assert not calls()
ok(apply()); ok(apply(y=out + y_bytes)); ok(apply(x=at, out=at + x_bytes)); ok(apply(y=out + 1024 + 2, out=out + 2))
assert len([c for c in calls() if c.startswith("launch")]) == 4
for h in (past, who): lib.kc_adapter_rows_free(h)
lib.kc_adapters_free(bank); lib.kc_adapters_free(None); lib.kc_adapter_rows_free(None)
assert lib.kc_live_objects() == before
""")


def test_adapters_are_made_and_set_outside_captures(graphs):
    """Inside one the fill that empties a new bank's slots and the copies into one would be the graph's, not the call's."""
    run(graphs, """
bank, who = C.c_void_p(), C.c_void_p()
slots = (C.c_int32 * 3)(0, -1, 1)
def make():
    b, r = C.c_void_p(), C.c_void_p()
    return lib.kc_adapters_create(ctx, 64, 48, 3, 20, C.byref(b)), lib.kc_adapter_rows_create(ctx, slots, 3, C.byref(r)), b, r
rc, rc_rows, bank, who = make()
ok(rc); ok(rc_rows)
def put():
    return lib.kc_adapters_set(bank, 1, at, at, 20, 1.0, 0), lib.kc_adapters_set(bank, 1, None, None, 0, 0.0, 0)
before = lib.kc_live_objects()
fake.fake_reset()
fake.fake_capture(1)
assert put() == (L.KC_ERR_INVALID, L.KC_ERR_INVALID) and b"captured" in lib.kc_last_error()
rc, rc_rows, b, r = make()
assert rc == rc_rows == L.KC_ERR_INVALID and not b.value and not r.value and lib.kc_live_objects() == before
assert not calls()
ok(lib.kc_adapters_apply(bank, who, at, at + 4096, at + 4096))     # the product may be captured
fake.fake_capture(0)
assert put() == (0, 0)
rc, rc_rows, b, r = make()
ok(rc); ok(rc_rows)
for h in (r, who): lib.kc_adapter_rows_free(h)
for h in (b, bank): lib.kc_adapters_free(h)
""")


SHARED = """
ok(lib.kc_kv_create(ctx, 1, 8, 128, 400, 16, L.KC_BF16, C.byref(kv)))
def behind(prefix, tails):
    seqs, free = [], prefix // 16
    for t in tails:
        n = -(-(prefix + t + 1) // 16) - prefix // 16
        ids = list(range(prefix // 16)) + list(range(free, free + n))
        free += n
        seqs.append((prefix + t, (C.c_uint32 * len(ids))(*ids)))
    return (L.KcSeqStep * len(seqs))(*[L.KcSeqStep(1, off, 1, len(b), b) for off, b in seqs])
tails = [3 + i for i in range(48)]
seqs = behind(4096, tails)          # 48 x 32 heads x 9 chunks of 520 bytes: 7 MB
"""


def test_a_plan_without_memory_for_sharing(graphs):
    """Sequences whose own units need no workspace are planned apart where the one for sharing is refused, with and without the margin."""
    run(graphs, SHARED + """
read, apart = C.c_int64(), C.c_int64()
p = C.c_void_p()
def shares():
    ok(lib.kc_attn_plan_keys(p, C.byref(read), C.byref(apart)))
    assert apart.value == sum(4096 + t + 1 for t in tails)
    ok(lib.kc_attn_plan_run(p, 0, at, 0.1, 0.0, 0, at + (1 << 19)))
    ok(lib.kc_attn_plan_run(p, 0, at, 0.1, 50.0, 0, at + (1 << 19)))
    return read.value < apart.value
fake.fake_fail_above(1 << 20)
ok(lib.kc_attn_plan_create(ctx, kv, seqs, 48, 32, C.byref(p)))
fake.fake_reset()
assert not shares()
assert calls() == ["launch in order"] * 2
ok(lib.kc_attn_plan_set(p, seqs, 48))
assert not shares() and "malloc" not in calls()   # not asked again at once
fake.fake_fail_above(2 ** 62)
for i in range(300):
    ok(lib.kc_attn_plan_set(p, seqs, 48))
assert shares() and calls().count("malloc") == 1
lib.kc_attn_plan_free(p)
fake.fake_fail_above(8 << 20)                     # room for what it needs
ok(lib.kc_attn_plan_create(ctx, kv, seqs, 48, 32, C.byref(p)))
assert shares()
lib.kc_attn_plan_free(p)
""")


def test_a_step_without_memory_for_sharing(graphs):
    """Forward, verify and decode steps run with the units that they would have without sharing."""
    run(graphs, SHARED + """
import dataclasses
import numpy as np
from kiln_b200 import api
from kiln_b200.synth import PRESETS, synth_checkpoint
fake.fake_shapes.restype = C.c_char_p
cfg = dataclasses.replace(PRESETS["tiny-llama"], num_attention_heads=32, num_key_value_heads=8, head_dim=128, num_hidden_layers=1)
c = api.Context(0)
model = api.CudaModel(c, cfg, synth_checkpoint(cfg, seed=0), max_step_tokens=64, max_step_seqs=48)
pool = api.PagedKv(c, model.kv_spec(400, 16))
ids, feed, out = (C.c_uint32 * 48)(), (C.c_int32 * 48)(*[-1] * 48), (C.c_uint32 * 48)()
logits, n, ticket, counts = C.c_void_p(), C.c_int32(), C.c_uint64(), (C.c_int32 * 48)()
lib = L.lib()
lib.kc_decode_launch.argtypes = L._SIGNATURES["kc_decode_launch"][1]
def steps():
    yield lib.kc_forward_step(model._h, pool._h, ids, 48, seqs, 48, 0, C.byref(logits), C.byref(n))
    yield lib.kc_verify_step(model._h, pool._h, ids, 48, seqs, 48, out, counts, counts)
    yield lib.kc_decode_launch(model._h, pool._h, ids, feed, seqs, 48, C.byref(ticket))
def attention():
    grids = []
    for rc in steps():
        assert rc == 0, lib.kc_last_error()
        grids.append([s for s in fake.fake_shapes().decode().split() if s.split(":")[0] in ("384", "768")])
        fake.fake_reset()
    return grids
fake.fake_fail_above(1 << 20)
refused = attention()
fake.fake_fail_above(2 ** 62)
for _ in range(100): attention()
shared = attention()
assert refused[0] == refused[1] == refused[2] and shared[0] == shared[1] == shared[2] != refused[0], (refused, shared)
""", first="import torch")


@pytest.mark.parametrize("heads,kv_heads,hd,rows,k,prefix,others,length,capped,shared", [
    (32, 8, 128, 5, 3, 8192, 125, 4096, False, False), (64, 8, 128, 5, 8, 4096, 100, 2048, False, False), (16, 8, 256, 1, 40, 1648, 81, 5088, True, False),
    (32, 8, 128, 1, 3, 8192, 125, 4096, False, False), (28, 4, 128, 1, 8, 8192, 60, 4096, False, True), (32, 8, 128, 1, 16, 2048, 48, 2048, False, True),
    (32, 8, 128, 5, 48, 4096, 0, 0, False, True), (32, 8, 128, 1, 48, 4096, 1, 60000, False, True), (64, 8, 128, 5, 64, 4096, 0, 0, False, True),
    (32, 8, 64, 1, 64, 6001, 0, 0, False, True), (16, 8, 256, 4, 16, 6144, 0, 0, True, True)])
def test_a_few_that_share_among_many(graphs, heads, kv_heads, hd, rows, k, prefix, others, length, capped, shared):
    """Chunks read together make units of one chunk of every other sequence too: where few of a step share, what it costs the
    others is weighed against it. Such steps were measured both ways, 7 % and more apart."""
    run(graphs, f"""
ok(lib.kc_kv_create(ctx, 1, {kv_heads}, {hd}, 6000, 16, L.KC_BF16, C.byref(kv)))
full, tail, seqs, tables = {prefix} // 16, 40, [], []
for i in range({k}):
    n = -(-({prefix} + tail + {rows}) // 16) - full
    tables.append((C.c_uint32 * (full + n))(*range(full), *(full + i * n + b for b in range(n))))
    seqs.append(L.KcSeqStep({rows}, {prefix} + tail, 0, full + n, tables[-1]))
for i in range({others}):                          # tables that agree nowhere
    n = -(-({length} + {rows}) // 16)
    tables.append((C.c_uint32 * n)(*((b + 7 * i) % 4000 + 2000 for b in range(n))))
    seqs.append(L.KcSeqStep({rows}, {length}, 0, n, tables[-1]))
p, read, apart = C.c_void_p(), C.c_int64(), C.c_int64()
ok(lib.kc_attn_plan_create(ctx, kv, (L.KcSeqStep * len(seqs))(*seqs), len(seqs), {heads}, C.byref(p)))
ok(lib.kc_attn_plan_keys(p, C.byref(read), C.byref(apart)))
fake.fake_reset()
ok(lib.kc_attn_plan_run(p, 0, at, 0.1, {50.0 if capped else 0.0}, 0, at + (1 << 19) * {1 if rows * (k + others) * heads * hd * 2 <= 1 << 19 else 100}))
launched = len([c for c in calls() if c.startswith("launch")])
if not {capped}: assert (read.value < apart.value) == {shared}, (read.value, apart.value)
assert (launched > 1) == {shared}, launched
""")


@pytest.mark.parametrize("sample_rows", [-1, 0, 3, 4, 2 ** 31 - 1])
def test_a_plan_samples_nothing(graphs, sample_rows):
    """sample_rows have no say in a plan: neither in whether it is taken nor in what it holds."""
    run(graphs, f"""
p = C.c_void_p()
seqs = (L.KcSeqStep * 2)(L.KcSeqStep(3, 40, {sample_rows}, 3, table), L.KcSeqStep(1, 7, {sample_rows}, 1, table))
ok(lib.kc_attn_plan_create(ctx, kv, seqs, 2, 4, C.byref(p)))
ok(lib.kc_attn_plan_set(p, seqs, 2))
assert seqs[0].sample_rows == seqs[1].sample_rows == {sample_rows}
ok(lib.kc_attn_plan_run(p, 0, at, 0.1, 0.0, 0, at + 4096))
lib.kc_attn_plan_free(p)
""")


@pytest.mark.parametrize("heads,kv_heads,hd,rows,k,prefix,launches", [
    (64, 8, 64, 8, 108, 2432, 2), (64, 8, 128, 8, 173, 2448, 2), (32, 8, 64, 1, 128, 6001, 3), (32, 8, 128, 4, 250, 2448, 3)])
def test_a_chunk_in_part_is_gone_on_from_where_the_kernel_is_the_faster_one(graphs, heads, kv_heads, hd, rows, k, prefix, launches):
    """The launch that goes on from the shared pieces of a chunk is of the kernel with a key per thread; where a step's own
    units take the other one, a chunk that is shared in part is each sequence's own."""
    run(graphs, f"""
ok(lib.kc_kv_create(ctx, 1, {kv_heads}, {hd}, 6000, 16, L.KC_BF16, C.byref(kv)))
full, seqs, tables = {prefix} // 16, [], []
for i in range({k}):
    n = -(-({prefix} + 40 + {rows}) // 16) - full
    tables.append((C.c_uint32 * (full + n))(*range(full), *(full + i * n + b for b in range(n))))
    seqs.append(L.KcSeqStep({rows}, {prefix} + 40, 0, full + n, tables[-1]))
p = C.c_void_p()
ok(lib.kc_attn_plan_create(ctx, kv, (L.KcSeqStep * len(seqs))(*seqs), len(seqs), {heads}, C.byref(p)))
fake.fake_reset()
ok(lib.kc_attn_plan_run(p, 0, at, 0.1, 0.0, 0, at + (1 << 28)))
assert len([c for c in calls() if c.startswith("launch")]) == {launches}
""")


@pytest.mark.parametrize("heads,kv_heads,hd,rows,k,prefix,others,length,shared", [
    (28, 4, 128, 8, 211, 896, 49, 74, False), (64, 8, 128, 8, 89, 1424, 180, 706, False), (64, 8, 128, 8, 219, 896, 0, 0, False),
    (64, 8, 128, 8, 173, 2448, 0, 0, True), (64, 8, 64, 8, 108, 2432, 0, 0, True)])
def test_partial_results_of_many_rows(graphs, heads, kv_heads, hd, rows, k, prefix, others, length, shared):
    """Rows of wide groups: what they leave for a chunk and what is merged is as much as the chunk's keys. Measured both ways, 8 % and
    more apart."""
    run(graphs, f"""
ok(lib.kc_kv_create(ctx, 1, {kv_heads}, {hd}, 6000, 16, L.KC_BF16, C.byref(kv)))
full, seqs, tables = {prefix} // 16, [], []
for i in range({k}):
    n = -(-({prefix} + 40 + {rows}) // 16) - full
    tables.append((C.c_uint32 * (full + n))(*range(full), *(full + i * n + b for b in range(n))))
    seqs.append(L.KcSeqStep({rows}, {prefix} + 40, 0, full + n, tables[-1]))
for i in range({others}):                          # tables that agree nowhere
    n = -(-({length} + {rows}) // 16)
    tables.append((C.c_uint32 * n)(*((b + 7 * i) % 2000 + 4000 for b in range(n))))
    seqs.append(L.KcSeqStep({rows}, {length}, 0, n, tables[-1]))
p, read, apart = C.c_void_p(), C.c_int64(), C.c_int64()
ok(lib.kc_attn_plan_create(ctx, kv, (L.KcSeqStep * len(seqs))(*seqs), len(seqs), {heads}, C.byref(p)))
ok(lib.kc_attn_plan_keys(p, C.byref(read), C.byref(apart)))
assert (read.value < apart.value) == {shared}, (read.value, apart.value)
""")
