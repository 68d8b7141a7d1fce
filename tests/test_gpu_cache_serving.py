"""Sessions that go on after an eviction: the steps of the integration notes,
token by token, against a 64-bit record of what each position was given."""

import ctypes

import numpy as np
import pytest

from cache_attn_ref import attend, ptr, torch_types
from test_gpu_cache_attn import check, evict_reference, f64, shape_of, status_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_tokens_appended_where_evicted_positions_lay(cuda_lib, kind):
    """Prompt, weights, eviction in place, then tokens appended behind the kept rows, each a row of K, V, pos and a
    record of 0, and a second eviction: no position inherits what an earlier one at its row was given."""
    import torch
    heads, kv, d, ctx, n, budget, first, last, more = 8, 2, 64, 96, 90, 40, 4, 8, 30
    g, w, batch, scale = heads // kv, heads * d, 2, d ** -0.5
    qt, ct = torch_types(kind)
    gen = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s, t: torch.randn(*s, generator=gen, device="cuda").to(t)
    q = 1.5 * rnd(batch, n + more, w, t=qt)
    new_k, new_v = (rnd(batch, kv, n + more, d, t=ct) for _ in range(2))  # by original position
    k, v = (torch.zeros(batch, kv, ctx, d, dtype=ct, device="cuda") for _ in range(2))
    k[:, :, :n], v[:, :, :n] = new_k[:, :, :n], new_v[:, :, :n]
    acc = torch.zeros(batch, kv, ctx, device="cuda")
    pos = torch.arange(ctx, dtype=torch.int32, device="cuda").expand(batch, kv, ctx).contiguous()
    sh = shape_of(kind, heads, kv, d, ctx)
    out, lse = torch.zeros(n, w, dtype=qt, device="cuda"), torch.zeros(n, heads, device="cuda")
    step = torch.zeros(batch, w, dtype=qt, device="cuda")
    given = np.zeros((batch, kv, n + more))  # the weight that each original position was given
    q64, k64, v64 = f64(q.cpu()), f64(new_k.cpu()), f64(new_v.cpu())

    def note(s, t, at):
        """The query at original position t sees the original positions at[kv head]."""
        for h in range(heads):
            j = at[h // g]
            given[s, h // g, j] += attend(q64[s, t, h * d:(h + 1) * d], k64[s, h // g, j], v64[s, h // g, j],
                                          np.ones(len(j), bool), scale)[2]

    for s in range(batch):
        check(cuda_lib.lfm_attention_window(sh, ptr(q[s]), w, ptr(k[s]), ptr(v[s]), 0, n, 0, 0, ptr(out), w, ptr(lse),
                                            None), "window")
        check(cuda_lib.lfm_attention_weights(sh, ptr(q[s]), w, ptr(k[s]), 0, n, 0, 0, ptr(lse), ptr(acc[s]), None), "weights")
        for t in range(n):
            note(s, t, [np.arange(t + 1)] * kv)
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")

    def evict():
        """In place; the choice is the plain one of the record as it was, and the record is what was given."""
        m = int(lens[0])
        before, where = acc.cpu().numpy(), pos.cpu().numpy()
        for s in range(batch):
            for h in range(kv):
                want = given[s, h, where[s, h, :m]]
                # fp32 sums of weights that are off by a few fp32 steps of their scores (bf16: of the scores as given)
                assert np.abs(before[s, h, :m] - want).max() <= 1e-4 * max(1.0, want.max()), (s, h)
        lo = torch.zeros(batch, dtype=torch.int32, device="cuda")
        check(cuda_lib.lfm_cache_evict(sh, *map(ptr, (k, v, acc, pos)), *map(ptr, (k, v, acc, pos)), kv * ctx * d, batch,
                                       None, ptr(lens), ptr(lo), batch, ctx, budget, first, last, None), "evict")
        after = pos.cpu().numpy()
        for s in range(batch):
            for h in range(kv):
                keep = evict_reference(before[s, h], m, budget, first, last)
                assert after[s, h, :budget].tolist() == where[s, h, keep].tolist()
        lens.copy_(lo)
        assert lens.tolist() == [budget] * batch

    evict()
    for t in range(n, n + more):
        row = int(lens[0])  # a token is appended: K, V, what the row holds, and a record of 0
        k[:, :, row], v[:, :, row], pos[:, :, row], acc[:, :, row] = new_k[:, :, t], new_v[:, :, t], t, 0
        lens += 1
        qs = q[:, t].contiguous()
        check(cuda_lib.lfm_attention_decode(sh, ptr(qs), w, ptr(k), ptr(v), kv * ctx * d, batch, None, ptr(lens), batch, ctx,
                                            0, 0, ptr(acc), ptr(step), w, None), "decode")
        held = pos.cpu().numpy()[:, :, :row + 1]
        for s in range(batch):
            note(s, t, held[s])
    evict()
    assert status_of(cuda_lib) == 0
