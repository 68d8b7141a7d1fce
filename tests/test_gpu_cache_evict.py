"""Eviction from session caches where weights repeat, layouts interleave and
rows are next to others': whole arrays against the plain choice, bit for bit."""

import numpy as np
import pytest

from cache_attn_ref import ptr
from test_gpu_cache_attn import check, evict_reference, shape_of, status_of

pytestmark = pytest.mark.gpu


def weights_of(pattern, rng, n):
    """n weights whose order keys meet a warp's 32 neighbours in ways of their own."""
    at = np.arange(n)
    if pattern == "equal":
        return np.full(n, 0.25, np.float32)
    if pattern == "halves":  # 17 equal ones, then 15 different
        return np.where(at % 32 < 17, 0.5, rng.random(n)).astype(np.float32)
    if pattern == "pairs":
        return rng.permutation(n).astype(np.float32) // 2
    if pattern == "near":  # the same high bits, different low ones: every pass counts on
        return (1.0 + rng.integers(0, 1024, n) * 2.0 ** -23).astype(np.float32)
    return np.where(rng.random(n) < 0.7, 0.0, rng.random(n)).astype(np.float32)  # mostly never looked at


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pattern", ["equal", "halves", "pairs", "near", "zeros"])
@pytest.mark.parametrize("lens,budget,first,last", [([1, 31, 33, 65, 257], 30, 1, 2), ([2001, 1999, 777], 700, 3, 70),
                                                    ([9001], 4444, 4, 100)])
def test_weights_that_repeat(cuda_lib, lens, budget, first, last, pattern, in_place):
    import torch
    kv, d, batch, ctx = 2, 64, len(lens), max(lens) + 3
    rng = np.random.default_rng(sum(lens))
    acc = np.stack([[weights_of(pattern, rng, ctx) for _ in range(kv)] for _ in range(batch)])
    k, v = (rng.integers(-32768, 32767, (batch, kv, ctx, d), dtype=np.int16) for _ in range(2))
    pos = rng.integers(0, 1 << 30, acc.shape).astype(np.int32)
    src = [k, v, acc, pos]
    want = [x.copy() if in_place else np.full_like(x, 7) for x in src]
    for b, n in enumerate(lens):
        for h in range(kv):
            keep = evict_reference(acc[b, h], n, budget, first, last)
            for x, w in zip(src, want):
                w[b, h, :len(keep)] = x[b, h, keep]
    s = [torch.from_numpy(x).cuda() for x in src]
    o = s if in_place else [torch.full_like(x, 7) for x in s]
    ld, lo = torch.tensor(lens, dtype=torch.int32).cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda")
    check(cuda_lib.lfm_cache_evict(shape_of("f16", kv, kv, d, ctx), *map(ptr, s), *map(ptr, o), kv * ctx * d, batch, None,
                                   ptr(ld), ptr(lo), batch, max(lens), budget, first, last, None), "evict")
    assert status_of(cuda_lib) == 0
    assert lo.cpu().tolist() == [min(n, budget) for n in lens]
    for x, w in zip(o, want):
        assert np.array_equal(x.cpu().numpy(), w)
