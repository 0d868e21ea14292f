"""Borders of a drawn row that lie where sums of its masses are a rounding apart: the kernel adds the masses up to each run of binades
in a tree, whose sum behind a run without tokens may be a rounding above the total. No such sum may move a border or a token."""
import numpy as np
import pytest
import torch

from kiln_b200 import api

pytestmark = pytest.mark.gpu


def tree_sums(x):
    """Sums up to each of 32 lanes, added by lanes 1, 2, 4, 8 and 16 apart."""
    x = x.copy()
    for o in (1, 2, 4, 8, 16):
        y = x.copy()
        y[:, o:] = x[:, o:] + x[:, :-o]
        x = y
    return x


def three_runs(rows, vocab, seed):
    """Rows with positive values, zeros and negative ones, most of them near 0 (the masses of all three runs count)."""
    rng = np.random.default_rng(seed)
    return np.round(rng.normal(0, 1, (rows, vocab)) * 32) / 32


def last_kept(row, top_k):
    order = np.argsort(-(row + 0.0), kind="stable")
    return order[min(top_k, len(row)) - 1 if top_k > 0 else -1]


def test_the_rows_have_such_sums():
    """What the next test is about: positive values are lane 4, zeros 9, negative ones 14; those behind 14 are empty."""
    x = three_runs(4000, 203, 1)
    w = np.exp(x - x.max(1, keepdims=True))
    lanes = np.zeros((len(x), 32))
    lanes[:, 4], lanes[:, 9], lanes[:, 14] = (w * (x > 0)).sum(1), (w * (x == 0)).sum(1), (w * (x < 0)).sum(1)
    sums = tree_sums(lanes)
    assert 100 < (sums[:, 15:19] > sums[:, 31:]).any(1).sum() < 2000


@pytest.mark.parametrize("u", [1.0, 1.5, float("inf"), float("nan")])
@pytest.mark.parametrize("rows", [30, 4000])      # eight CTAs a row; two, three on an SM
def test_one_and_more_is_the_last_token_kept(ctx, rows, u):
    x = three_runs(rows, 203, 1)
    settings = [(0, 0, 7, 100)[r % 4] for r in range(rows)]
    packed = api.pack_sampling([api.SamplingParams(1.0, k) for k in settings], "cuda")
    tokens, logprobs = api.sample_rows(ctx, torch.from_numpy(x).to(torch.bfloat16).cuda(), packed, torch.full((rows,), u, device="cuda"))
    want = [last_kept(r, k) for r, k in zip(x, settings)]
    assert tokens.tolist() == [int(t) for t in want]
    # half a step of fp32 of a value below 16, and what a share that is 1e-13 off loses
    for r in range(rows):
        order = np.sort(x[r])[::-1][: settings[r] or None]
        want = order[-1] - order[0] - np.log(np.exp(order - order[0]).sum())
        assert abs(float(logprobs[r]) - want) <= 16 * 2.0 ** -24 + 1e-12


@pytest.mark.parametrize("top_k", [0, 40])
def test_a_tail_without_weight(ctx, top_k):
    """Tokens whose weights are below the rounding of the sum, so that sums up to many of them are the total."""
    rng = np.random.default_rng(3)
    x = np.concatenate([np.full((64, 1), 60.0), rng.integers(-16, 17, (64, 300)) / 4], 1)
    tokens, _ = api.sample_rows(ctx, torch.from_numpy(x).to(torch.bfloat16).cuda(), [api.SamplingParams(1.0, top_k)] * 64, torch.ones(64, device="cuda"))
    assert tokens.tolist() == [int(last_kept(r, top_k)) for r in x]
