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
