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


@pytest.mark.parametrize("in_place", [False, True])
def test_keys_and_values_of_a_slot_side_by_side(cuda_lib, in_place):
    """One array [slot][K, V][kv][ctx][d]: the calls take K and V as two caches of twice the stride."""
    import torch
    n_slots, kv, ctx, d, lens, budget, first, last = 4, 2, 150, 64, [150, 91, 33], 40, 3, 10
    rng = np.random.default_rng(12)
    both = rng.integers(-32768, 32767, (n_slots, 2, kv, ctx, d), dtype=np.int16)
    acc = rng.random((n_slots, kv, ctx)).astype(np.float32)
    slots = [2, 0, 3]
    want, want_acc = both.copy() if in_place else np.full_like(both, 7), acc.copy() if in_place else np.full_like(acc, 7)
    for slot, n in zip(slots, lens):
        for h in range(kv):
            keep = evict_reference(acc[slot, h], n, budget, first, last)
            want[slot, :, h, :len(keep)] = both[slot][:, h, keep]
            want_acc[slot, h, :len(keep)] = acc[slot, h, keep]
    src = torch.from_numpy(both).cuda(), torch.from_numpy(acc).cuda()
    dst = src if in_place else tuple(torch.full_like(x, 7) for x in src)
    sd, ld = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (slots, lens))
    lo = torch.zeros(3, dtype=torch.int32, device="cuda")
    check(cuda_lib.lfm_cache_evict(shape_of("f16", kv, kv, d, ctx), ptr(src[0][:, 0]), ptr(src[0][:, 1]), ptr(src[1]), None,
                                   ptr(dst[0][:, 0]), ptr(dst[0][:, 1]), ptr(dst[1]), None, 2 * kv * ctx * d, n_slots,
                                   ptr(sd), ptr(ld), ptr(lo), 3, max(lens), budget, first, last, None), "evict")
    assert status_of(cuda_lib) == 0
    assert lo.cpu().tolist() == [40, 40, 33]
    assert np.array_equal(dst[0].cpu().numpy(), want) and np.array_equal(dst[1].cpu().numpy(), want_acc)
