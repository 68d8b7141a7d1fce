"""What the norm limits of the session-cache attention tests catch, on an
emulation of the kernels' number formats (no GPU)."""

import numpy as np
import pytest

from cache_attn_norm import SHIFT, dominated, emulate_f32, fp16_floor, limit, norm_error, plain32, score_cut
from cache_attn_ref import attend


def _errors(q, k, v, **kw):
    scale, every = q.shape[1] ** -0.5, np.ones(k.shape[1], bool)
    g = len(q) // len(k)
    rows = [attend(x, k[i // g], v[i // g], every, scale) for i, x in enumerate(q)]
    want = np.stack([r[0] for r in rows])
    floor = np.linalg.norm([fp16_floor(r[2], v[i // g], SHIFT["f32"]) for i, r in enumerate(rows)]) / np.linalg.norm(want)
    floor += max(score_cut(q.shape[1], k[i // g] @ x * scale) for i, x in enumerate(q))
    plain = np.stack([plain32(x, k[i // g], v[i // g], scale) for i, x in enumerate(q)])
    got = np.stack([emulate_f32(x, k[i // g], v[i // g], scale, **kw) for i, x in enumerate(q)])
    return norm_error(got, want), limit("f32", norm_error(plain, want), floor)


@pytest.mark.parametrize("nats", [6, 8, 10, 14])
def test_weights_relative_to_the_maximum_alone_are_caught(nats):
    q, k, v = dominated(np.random.default_rng(nats), "f32", 8, 2, 2000, 64, nats, 3)
    error, most = _errors(q, k, v)
    assert error <= most
    error, most = _errors(q, k, v, shift=0.0)
    assert error > 4 * most


@pytest.mark.parametrize("d,n", [(64, 1), (64, 40), (128, 577), (64, 4000)])
@pytest.mark.parametrize("lost", [{}, {"q_low": False}, {"p_low": False}])
def test_a_lost_half_of_a_pair_is_caught(d, n, lost):
    rng = np.random.default_rng(n)
    q, k, v = rng.normal(0, 1.5, (8, d)), rng.normal(0, 1, (2, n, d)), rng.normal(0, 1, (2, n, d))
    q, k, v = (x.astype(t).astype(np.float64) for x, t in ((q, np.float32), (k, np.float16), (v, np.float16)))
    error, most = _errors(q, k, v, **lost)
    if lost and n > 1:  # one position alone has weight 1, whatever its score
        assert error > 4 * most
    else:
        assert error <= most


@pytest.mark.parametrize("size", [1e-4, 1e-2])
def test_small_queries_that_are_not_brought_to_size_are_caught(size):
    rng = np.random.default_rng(3)
    q, k, v = rng.normal(0, size, (8, 64)), rng.normal(0, 1 / size, (2, 500, 64)), rng.normal(0, 1, (2, 500, 64))
    q, k, v = (x.astype(t).astype(np.float64) for x, t in ((q, np.float32), (k, np.float16), (v, np.float16)))
    error, most = _errors(q, k, v)
    assert error <= most
    error, most = _errors(q, k, v, to_size=False)
    assert error > 2 * most
