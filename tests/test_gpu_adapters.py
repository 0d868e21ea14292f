"""Low-rank adapters beside a projection against the formula in 64 bits. The result is rounded to bf16 once: half a step of its value
(2^-8 of it at the most), and the fp32 sums before that: a term of A x or B t is off by 2^-24 of the sum of their absolute values
for each of the additions, and t = A x, scaled, goes into the second product as a bf16 number: off by half a step, 2^-8 of it at the most."""
import numpy as np
import pytest
import torch

from kiln_b200 import api
from kiln_b200.synth import quantize_affine

pytestmark = pytest.mark.gpu


def bank(ctx, n_in, n_out, ranks, seed, max_rank=None, std=0.1):
    g = torch.Generator().manual_seed(seed)
    ad = api.Adapters(ctx, n_in, n_out, len(ranks), max_rank or max(ranks))
    parts = []
    for i, r in enumerate(ranks):
        a, b = (torch.empty(s).normal_(0, d, generator=g).to(torch.bfloat16) for s, d in (((r, n_in), n_in ** -0.5), ((n_out, r), std)))
        scale = [1.0, 0.5, -2.0][i % 3]
        ad.set(i, a.cuda() if i % 2 else a, b.cuda() if i % 2 else b, scale)
        parts.append((a.cuda().double(), b.cuda().double(), scale))
    return ad, parts


def inputs(m, n_in, n_out, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.empty(m, n, device="cuda").normal_(generator=g).to(torch.bfloat16) for n in (n_in, n_out)]


def formula(parts, x, y, slots):
    """The result in 64 bits and what its fp32 sums may be off by."""
    out, off = y.double(), torch.zeros_like(y, dtype=torch.float64)
    for i, (a, b, scale) in enumerate(parts):
        rows = torch.from_numpy(np.flatnonzero(np.asarray(slots) == i)).cuda()
        if len(rows):
            v = x[rows].double()
            t, t_abs = v @ a.T, v.abs() @ a.abs().T
            out[rows] += scale * (t @ b.T)
            n_in, rank = a.shape[1], a.shape[0]
            off[rows] = abs(scale) * ((t_abs * (n_in * 2.0 ** -24)) @ b.abs().T + t.abs() @ b.abs().T * (2.0 ** -8 + (2 * rank + 2) * 2.0 ** -24))
    return out, off


def check(got, want, off):
    d = (got.double() - want).abs()
    assert bool((d <= want.abs() * 2.0 ** -8 + off * 1.01 + 1e-30).all()), float((d - want.abs() * 2.0 ** -8 - off).max())


@pytest.mark.parametrize("n_in,n_out", [(32, 1), (64, 8), (64, 40), (96, 31), (2048, 520), (4096, 4096), (3584, 1001), (224, 2050)])
@pytest.mark.parametrize("ranks", [[1], [16, 3], [8, 17, 32], [64, 1, 33, 64], [128, 5, 96, 100]])
def test_rows_take_their_adapters(ctx, n_in, n_out, ranks):
    ad, parts = bank(ctx, n_in, n_out, ranks, n_in + n_out)
    for m in (1, 2, 15, 16, 17, 33, 70):
        rng = np.random.default_rng(m)
        slots = rng.integers(-1, len(ranks), m)
        x, y = inputs(m, n_in, n_out, m)
        want, off = formula(parts, x, y, slots)
        rows = api.AdapterRows(ctx, slots)
        got = ad.apply(x, rows, y)
        torch.cuda.synchronize()
        check(got, want, off)
        none = torch.from_numpy(slots < 0).cuda()
        assert torch.equal(got[none], y[none])
        assert ad.apply(x, rows, y, out=y) is y                    # in place: the same bits
        torch.cuda.synchronize()
        assert torch.equal(got, y)


@pytest.mark.parametrize("m,used", [(64, 1), (65, 1), (300, 2), (1000, 3), (2048, 8), (2050, 1)])
def test_many_rows(ctx, m, used):
    """Tiles of 16 rows, the last ones in part; every row once."""
    ad, parts = bank(ctx, 256, 264, [24] * used, m)
    slots = np.sort(np.random.default_rng(m).integers(0, used, m))
    x, y = inputs(m, 256, 264, m)
    want, off = formula(parts, x, y, slots)
    got = ad.apply(x, api.AdapterRows(ctx, slots), y)
    torch.cuda.synchronize()
    check(got, want, off)


def test_a_row_does_not_hang_on_the_others(ctx):
    """The same bits alone, among others in another order, and in tiles of another size."""
    ad, _ = bank(ctx, 1024, 1032, [40, 64, 16], 1)
    rng = np.random.default_rng(1)
    slots = rng.integers(-1, 3, 900)
    x, y = inputs(900, 1024, 1032, 2)
    all_rows = ad.apply(x, api.AdapterRows(ctx, slots), y)
    order = rng.permutation(900)[:50]
    some = ad.apply(x[order].contiguous(), api.AdapterRows(ctx, slots[order]), y[order].contiguous())
    torch.cuda.synchronize()
    assert torch.equal(some, all_rows[torch.from_numpy(order).cuda()])


@pytest.mark.parametrize("n_in,n_out,rank", [(96, 41, 16), (1024, 1032, 30), (1024, 520, 64), (2080, 264, 128)])
def test_every_size_of_cluster(ctx, n_in, n_out, rank):
    """Tiles by the dozen and by the hundred, whose clusters have eight to two CTAs: a row's bits are the same in all."""
    ad, parts = bank(ctx, n_in, n_out, [rank] * 3, 1)
    x, y = inputs(16 * 150, n_in, n_out, 2)
    slots = np.repeat(np.arange(150) % 3, 16)
    want, off = formula(parts, x, y, slots)
    before = None
    for tiles in (1, 8, 16, 17, 18, 20, 21, 33, 35, 36, 40, 42, 45, 47, 60, 72, 85, 90, 93, 150):
        n = 16 * tiles
        got = ad.apply(x[:n], api.AdapterRows(ctx, slots[:n]), y[:n])
        torch.cuda.synchronize()
        assert before is None or torch.equal(got[: before.shape[0]], before)
        before = got
    check(got, want, off)


@pytest.mark.parametrize("shift", [1, 3, 4, 8])
def test_rows_off_16_byte_boundaries(ctx, shift):
    """y and out that start anywhere; what lies around out is left."""
    ad, parts = bank(ctx, 64, 48, [8], 3)
    x, y = inputs(5, 64, 48, 1)
    want, off = formula(parts, x, y, [0] * 5)
    room = torch.full((5 * 48 + 16,), 9.0, dtype=torch.bfloat16, device="cuda")
    out = room[shift: shift + 240].view(5, 48)
    there = torch.zeros(5 * 48 + 16, dtype=torch.bfloat16, device="cuda")[shift: shift + 240].view(5, 48)
    there.copy_(y)
    ad.apply(x, api.AdapterRows(ctx, [0] * 5), there, out=out)
    torch.cuda.synchronize()
    check(out, want, off)
    assert (room[:shift] == 9).all() and (room[shift + 240:] == 9).all()


def test_infinities_stay_in_their_rows(ctx):
    """An infinite or NaN activation has no say in other rows, and none through the zeros behind a slot's rank."""
    ad, parts = bank(ctx, 64, 16, [3, 3], 5, max_rank=32)
    x, y = inputs(20, 64, 16, 1)
    x[3, 5], x[9, 1] = float("inf"), float("nan")
    slots = [0] * 12 + [1] * 8
    got = ad.apply(x, api.AdapterRows(ctx, slots), y)
    x[3], x[9] = 0, 0
    want, off = formula(parts, x, y, slots)
    torch.cuda.synchronize()
    keep = [i for i in range(20) if i not in (3, 9)]
    check(got[keep], want[keep], off[keep])
    assert bool(got[9].isnan().all())
    t = parts[0][0][:, 5].sign() * float("inf")                    # what the infinite feature makes of row 3
    sums = torch.stack([torch.where(parts[0][1][:, r] == 0, torch.nan, parts[0][1][:, r] * t[r]) for r in range(3)]).sum(0)
    assert torch.equal(got[3].isnan(), sums.isnan()) and torch.equal(got[3][~sums.isnan()].double(), sums[~sums.isnan()])


def test_slots_are_replaced_and_emptied(ctx):
    ad, parts = bank(ctx, 128, 64, [16, 16], 7, max_rank=48)
    x, y = inputs(6, 128, 64, 2)
    rows = api.AdapterRows(ctx, [0, 1, 0, 1, -1, 0])
    other = api.Adapters(ctx, 128, 64, 4, 48)                      # never set: nothing is added
    assert torch.equal(other.apply(x, rows, y), y)
    a, b = (torch.randn(s).to(torch.bfloat16) for s in ((40, 128), (64, 40)))
    for new in ((a, b), (a[:5], b[:, :5])):                        # a larger rank, then a smaller one over it
        ad.set(0, *new, scale=0.25)
        parts[0] = (new[0].cuda().double(), new[1].cuda().double(), 0.25)
        want, off = formula(parts, x, y, [0, 1, 0, 1, -1, 0])
        got = ad.apply(x, rows, y)
        torch.cuda.synchronize()
        check(got, want, off)
    ad.clear(0)
    got = ad.apply(x, rows, y)
    torch.cuda.synchronize()
    assert torch.equal(got[[0, 2, 4, 5]], y[[0, 2, 4, 5]]) and not torch.equal(got[1], y[1])


def test_beside_a_quantised_projection(ctx):
    """QuantizedWeight.matmul with adapters is its product and what they add, in bf16 each."""
    g = torch.Generator().manual_seed(1)
    w, s, b = quantize_affine(torch.empty(1030, 512).normal_(0, 0.02, generator=g), 4, 64)
    weight = api.QuantizedWeight(ctx, w, s, b, 4, 64)
    ad, parts = bank(ctx, 512, 1030, [16, 8], 3)
    slots = [0, 1, -1, 0, 1, 1, 0]
    rows = api.AdapterRows(ctx, slots)
    x, _ = inputs(7, 512, 1030, 1)
    plain = weight.matmul(x)
    got = weight.matmul(x, ad, rows)
    check(got, *formula(parts, x, plain, slots))
    for bad in (dict(adapters=ad), dict(adapters=ad, rows=api.AdapterRows(ctx, slots[:3])), dict(adapters=api.Adapters(ctx, 512, 64, 1, 4), rows=rows)):
        with pytest.raises(ValueError):
            weight.matmul(x, **bad)
    with pytest.raises(ValueError):
        weight.matmul(x, rows=rows)
    ad.close()
    with pytest.raises(api.KcError):
        weight.matmul(x, ad, rows)
    assert torch.equal(weight.matmul(x), plain)


def test_streams_and_graphs(ctx):
    ad, _ = bank(ctx, 256, 512, [16, 32], 3)
    rows = api.AdapterRows(ctx, [0, 1, 1, -1, 0])
    x, y = inputs(5, 256, 512, 1)
    x2, y2 = inputs(5, 256, 512, 2)
    want, want2 = ad.apply(x, rows, y).clone(), ad.apply(x2, rows, y2).clone()
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.ExternalStream(ctx.stream)):
        with torch.cuda.stream(stream):
            u, v = torch.empty_like(x), torch.empty_like(y)
            for _ in range(20):
                u.copy_(x2); v.copy_(y2)
                a = ad.apply(u, rows, v)
                u.copy_(x); v.copy_(y)
                b = ad.apply(u, rows, v)
        torch.cuda.synchronize()
        assert torch.equal(a, want2) and torch.equal(b, want)
    u, v, out = x.clone(), y.clone(), torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ad.apply(u, rows, v, out=out)
    for p, q, w in ((x2, y2, want2), (x, y, want)):
        u.copy_(p); v.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    ctx.sync()


def test_a_slot_is_set_behind_a_graph_in_flight(ctx):
    """A replay on another stream than the context's, still to run when the host sets or empties the slot, has the slot as it was."""
    ad, parts = bank(ctx, 256, 512, [16, 16], 3)
    _, others = bank(ctx, 256, 512, [16, 16], 4)
    rows = api.AdapterRows(ctx, [0, 1, 1, -1, 0])
    x, y = inputs(5, 256, 512, 1)
    first = ad.apply(x, rows, y)
    out = torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ad.apply(x, rows, y, out=out)
    stream = torch.cuda.Stream()
    on_host = [t.to(torch.bfloat16).cpu() for t in others[0][:2]]
    changes = [lambda: ad.set(0, *on_host), lambda: ad.set(0, *(t.cuda() for t in on_host)), lambda: ad.clear(0)]
    for change in changes:
        ad.set(0, *(t.to(torch.bfloat16) for t in parts[0][:2]), parts[0][2])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out.zero_()
            torch.cuda._sleep(100_000_000)                         # some 50 ms
            graph.replay()
            change()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        graph.replay()
        torch.cuda.synchronize()
        assert not torch.equal(out, first)
        assert torch.equal(out, ad.apply(x, rows, y))


def test_a_slot_is_not_set_in_a_capture(ctx):
    """Refused, and the capture is what it would be without."""
    ad, parts = bank(ctx, 256, 512, [16, 16], 3)
    rows = api.AdapterRows(ctx, [0, 1, 1, -1, 0])
    x, y = inputs(5, 256, 512, 1)
    want, out = ad.apply(x, rows, y), torch.empty_like(y)
    a, b = (t.to(torch.bfloat16).cpu() for t in parts[1][:2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(api.KcError):
            ad.set(0, a, b)
        ad.apply(x, rows, y, out=out)
        with pytest.raises(api.KcError):
            ad.clear(0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals(ctx):
    live = api.live_objects()
    for n_in, n_out, slots, rank in ((31, 8, 1, 4), (0, 8, 1, 4), (48, 8, 1, 4), (64, 0, 1, 4), (64, 8, 0, 4), (64, 8, 1, 0), (64, 8, 1, 129)):
        with pytest.raises(api.KcError):
            api.Adapters(ctx, n_in, n_out, slots, rank)
    ad, _ = bank(ctx, 64, 8, [4, 4], 1)
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 4, dtype=torch.bfloat16)
    for slot, rank, scale in ((-1, 4, 1.0), (2, 4, 1.0), (0, 4, float("nan")), (0, 4, float("inf"))):
        with pytest.raises(api.KcError):
            ad.set(slot, a[:rank], b[:, :rank], scale)
    with pytest.raises(api.KcError):
        ad.set(0, torch.zeros(5, 64, dtype=torch.bfloat16), torch.zeros(8, 5, dtype=torch.bfloat16))
    for bad in ((a.float(), b.float()), (a[:, :32], b), (a, b.t()), (a.cuda(), b)):
        with pytest.raises(ValueError):
            ad.set(0, *bad)
    for slots in ([], [-2], [0, -5]):
        with pytest.raises(api.KcError):
            api.AdapterRows(ctx, slots)
    with pytest.raises(ValueError):
        api.AdapterRows(ctx, [[0, 1]])
    x, y = inputs(2, 64, 8, 1)
    rows = api.AdapterRows(ctx, [0, 2])
    with pytest.raises(api.KcError):
        ad.apply(x, rows, y)                                       # slot 2 of 2
    rows = api.AdapterRows(ctx, [0, 1])
    for bad in (dict(x=x.float()), dict(x=x[:1]), dict(y=y[:, :4]), dict(out=y.t()), dict(x=x.cpu()), dict(y=y.float())):
        with pytest.raises(ValueError):
            ad.apply(**{**dict(x=x, rows=rows, y=y), **bad})
    with pytest.raises(api.KcError):                               # x off a 16-byte boundary
        ad.apply(torch.zeros(130, dtype=torch.bfloat16, device="cuda")[1:129].view(2, 64), rows, y)
    second = api.Context(0)
    with pytest.raises(api.KcError):
        ad.apply(x, api.AdapterRows(second, [0, 1]), y)
    second.close()
    ad.close()
    with pytest.raises(api.KcError):
        ad.apply(x, rows, y)
    rows.close()
    assert api.live_objects() == live
