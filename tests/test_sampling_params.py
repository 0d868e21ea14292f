"""Settings and calls that are refused before anything reaches a device. Needs no GPU."""
import math

import numpy as np
import pytest

from kiln_b200 import _lib as L
from kiln_b200 import api
from tests.test_host_calls import fake, run  # noqa: F401  (a fixture)


@pytest.mark.parametrize("bad", [dict(temperature=-0.1), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_k=-1), dict(top_k=1 << 31), dict(top_p=0.0),
                                 dict(top_p=1.1), dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=math.nan)])
def test_settings_outside_their_range(bad):
    with pytest.raises(ValueError):
        api.SamplingParams(**bad)


def test_packed_settings_are_the_structs():
    t = api.pack_sampling([api.SamplingParams(0.5, 40, 0.9, 0.05), api.SamplingParams()], "cpu")
    want = (L.KcSampling * 2)(L.KcSampling(0.5, 40, 0.9, 0.05), L.KcSampling(1.0, 0, 1.0, 0.0))
    assert t.shape == (2, 4) and bytes(t.numpy().tobytes()) == bytes(want)
    assert api.pack_sampling([], "cpu").shape == (0, 4)


def test_random_numbers_stay_below_one():
    u = api._uniforms([0.0, 0.25, 1 - 2.0 ** -53, 1 - 2.0 ** -24, 1.0, -1.0, math.nan])
    assert u.dtype == np.float32 and u.tolist()[:6] == [0.0, 0.25, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1.0, -1.0] and math.isnan(u[6])
    assert api._uniforms([]).shape == (0,)


def test_calls_are_refused_before_a_launch(fake):  # noqa: F811
    run(fake, """
fake.fake_reset()
def sample(logits=at, ld=100, rows=2, vocab=100, sampling=at, u=at, tokens=at, logprobs=at):
    return lib.kc_sample_rows(ctx, logits, ld, rows, vocab, sampling, u, tokens, logprobs)
for bad in (dict(logits=None), dict(sampling=None), dict(u=None), dict(tokens=None), dict(rows=0), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(ld=-100),
            dict(vocab=(1 << 30) + 1, ld=1 << 40), dict(logits=at + 1), dict(sampling=at + 8), dict(u=at + 2), dict(tokens=at + 1), dict(logprobs=at + 3)):
    assert sample(**bad) == L.KC_ERR_INVALID, bad
    assert lib.kc_last_error()
assert lib.kc_sample_rows(None, at, 100, 2, 100, at, at, at, at) == L.KC_ERR_INVALID
assert not [c for c in calls() if c.startswith("launch")]
ok(sample()); ok(sample(logprobs=None)); ok(sample(rows=1, ld=0)); ok(sample(logits=at + 2, ld=101))
assert len([c for c in calls() if c.startswith("launch")]) == 4
""")


def test_settings_that_float32_does_not_have():
    """Positive and finite settings stay that: 0 and infinity have meanings of their own, and the verify round refuses a top_p of 0."""
    tiny, large = float(np.finfo(np.float32).smallest_subnormal), float(np.finfo(np.float32).max)
    got = api.pack_sampling([api.SamplingParams(1e-60, 0, 1e-46, 1e-300), api.SamplingParams(1e39), api.SamplingParams(0.0), api.SamplingParams(0.1, 3, 0.2, 0.3)], "cpu")
    f = got.numpy().view(np.float32)
    assert f[:, [0, 2, 3]].tolist() == [[tiny, tiny, tiny], [large, 1.0, 0.0], [0.0, 1.0, 0.0], [float(np.float32(x)) for x in (0.1, 0.2, 0.3)]]
    assert got[:, 1].tolist() == [0, 0, 0, 3]
