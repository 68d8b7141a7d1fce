"""Attention over session caches (lfm_attention_*, lfm_cache_evict) against
64-bit plain forms, at the sizes and masks where each can go wrong.

Every comparison's tolerance comes from the inputs by the error bounds of
cache_attn_ref (no constant is fitted)."""

import ctypes

import numpy as np
import pytest

from cache_attn_ref import TYPES, attend, out_error, ptr, score_error, seen, torch_types

pytestmark = pytest.mark.gpu


def shape_of(kind, heads, kv, d, ctx, scale=0.0):
    import lfm2_b200
    return lfm2_b200.AttnShape(TYPES[kind], heads, kv, d, ctx, scale)


def check(status, what):
    import lfm2_b200
    lfm2_b200.ops_check(status, what)


def status_of(lib):
    s = ctypes.c_uint32(99)
    check(lib.lfm_attention_status(ctypes.byref(s), None), "status")
    return s.value


def rows(rng, n, width, kind, stride, scale=1.0):
    """n rows of `width` values in rows of `stride`, the values behind them NaN."""
    import torch
    qt, _ = torch_types(kind)
    x = torch.full((n, stride), float("nan"), dtype=qt)
    x[:, :width] = torch.from_numpy(rng.normal(0, scale, (n, width))).to(qt)
    return x


def cache(rng, dims, kind):
    import torch
    _, ct = torch_types(kind)
    return torch.from_numpy(rng.normal(0, 1, dims)).to(ct)


def f64(t):
    import torch
    return t.to(torch.float64).numpy()


# ------------------------------------------------------------------- window
WINDOW = [  # kind, heads, kv, d, ctx, start, n, window, sinks, pad, scale
    ("f32", 32, 8, 64, 64, 0, 1, 0, 0, 0, 0.0),
    ("f32", 32, 8, 64, 512, 100, 64, 0, 0, 512, 0.0),
    ("f32", 32, 8, 64, 700, 0, 700, 100, 4, 512, 0.0),
    ("f32", 4, 1, 128, 333, 0, 333, 1, 0, 0, 0.0),
    ("f32", 24, 8, 64, 1300, 1200, 33, 128, 200, 4, 0.3),
    ("f16", 12, 2, 64, 260, 3, 257, 129, 1, 8, 0.0),
    ("f16", 8, 1, 128, 900, 0, 900, 256, 130, 0, 0.0),
    ("f16", 7, 7, 128, 130, 0, 130, 0, 3, 0, 0.0),
    ("bf16", 32, 4, 128, 640, 511, 129, 64, 5, 0, 0.0),
    ("bf16", 28, 4, 64, 1025, 1024, 1, 500, 7, 0, 0.0),
    ("bf16", 5, 1, 64, 400, 0, 400, 399, 1, 0, 0.5),
    ("bf16", 16, 8, 128, 300, 0, 300, 2000, 0, 8, 0.0),
]


def window_reference(kind, q, k, v, heads, kv, d, start, n, window, sinks, scale):
    out, lse, tol = np.zeros((n, heads * d)), np.zeros((n, heads)), np.zeros((n, heads * d))
    acc, tol_lse = np.zeros((kv, k.shape[1])), np.zeros((n, heads))
    for t in range(n):
        p = start + t
        see = seen(p, np.arange(p + 1), window, sinks)
        at = np.flatnonzero(see)
        for h in range(heads):
            kh = h // (heads // kv)
            qq = q[t, h * d:(h + 1) * d]
            o, e, w = attend(qq, k[kh, :p + 1], v[kh, :p + 1], see, scale)
            ds = score_error(kind, qq, k[kh, at], scale)
            out[t, h * d:(h + 1) * d], lse[t, h] = o, e
            acc[kh, :p + 1] += w
            tol[t, h * d:(h + 1) * d] = out_error(kind, ds, at.size, np.abs(v[kh, at]).max(), o)
            # the scores' error, the sum's (n + 8) steps, the logarithm's and the result's roundings
            tol_lse[t, h] = ds + (at.size + 16) * 2.0 ** -23 + 2.0 ** -22 * abs(e)
    return out, lse, acc, tol, tol_lse


@pytest.mark.parametrize("kind,heads,kv,d,ctx,start,n,window,sinks,pad,scale", WINDOW)
def test_window_and_weights(cuda_lib, kind, heads, kv, d, ctx, start, n, window, sinks, pad, scale):
    import torch
    rng = np.random.default_rng(heads * 1000 + n)
    width = heads * d
    q = rows(rng, n, width, kind, width + pad, 1.5)
    k, v = cache(rng, (kv, ctx, d), kind), cache(rng, (kv, ctx, d), kind)
    # what no query sees holds NaN: later positions, and those between the sinks and the first window
    unseen = np.ones(ctx, bool)
    for p in range(start, start + n):
        unseen[:p + 1] &= ~seen(p, np.arange(p + 1), window, sinks)
    k[:, unseen], v[:, unseen] = float("nan"), float("nan")
    sc = scale or d ** -0.5
    ref, lse_ref, acc_ref, tol, tol_lse = window_reference(
        kind, f64(q), f64(k), f64(v), heads, kv, d, start, n, window, sinks, sc)
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    out = torch.full((n + 1, width + 8), float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full((n + 1, heads), float("nan"), device="cuda")
    sh = shape_of(kind, heads, kv, d, ctx, scale)
    check(cuda_lib.lfm_attention_window(sh, ptr(qd), width + pad, ptr(kd), ptr(vd), start, n, window, sinks, ptr(out),
                                        width + 8, ptr(lse), None), "window")
    assert status_of(cuda_lib) == 0
    got = f64(out.cpu())
    assert np.isnan(got[:, width:]).all() and np.isnan(got[n]).all(), "wrote outside its rows"
    err = np.abs(got[:n, :width] - ref)
    assert (err <= tol).all(), (err.max(), (err / tol).max())
    lse_got = lse.cpu().double().numpy()
    assert np.isnan(lse_got[n]).all()
    err = np.abs(lse_got[:n] - lse_ref)
    assert (err <= tol_lse).all(), (err / tol_lse).max()
    # without the statistics: the same output
    out2 = torch.full_like(out, float("nan"))
    check(cuda_lib.lfm_attention_window(sh, ptr(qd), width + pad, ptr(kd), ptr(vd), start, n, window, sinks,
                                        ptr(out2), width + 8, None, None), "window")
    assert torch.equal(out2[:n, :width], out[:n, :width])

    # weights: given the exact statistics, added to what is there; the sum of n * group weights
    old = torch.rand(kv, ctx)
    accd = old.cuda()
    lse_in = torch.from_numpy(lse_ref).float().cuda()
    check(cuda_lib.lfm_attention_weights(sh, ptr(qd), width + pad, ptr(kd), start, n, window, sinks, ptr(lse_in),
                                         ptr(accd), None), "weights")
    assert status_of(cuda_lib) == 0
    got = accd.cpu().double().numpy()
    fits = ~unseen
    ds = max(score_error(kind, f64(q)[:, h * d:(h + 1) * d], f64(k)[h // (heads // kv)][fits], sc) for h in range(heads))
    # each term: its score's error, the statistics' rounding, the exponential's 2^-21; the sum's steps
    many = n * (heads // kv)
    rel = ds * (1 + ds) + np.abs(lse_ref).max() * 2.0 ** -23 + 2.0 ** -20 + (many + 4) * 2.0 ** -23
    want = acc_ref + old.double().numpy()
    err = np.abs(got - want)
    assert (err <= rel * acc_ref + 2.0 ** -23 * want).all(), (err.max(), ds)
    assert np.array_equal(got[:, unseen], old.double().numpy()[:, unseen])


def test_window_matches_the_engines_prompt_attention(cuda_lib):
    """Without a window and on the engine's layout both entry points give the same attention."""
    import torch
    rng = np.random.default_rng(5)
    n, ctx = 200, 256
    q = torch.from_numpy(rng.normal(0, 1, (n, 2048))).float().cuda()
    k, v = (torch.from_numpy(rng.normal(0, 1, (8, ctx, 64))).half().cuda() for _ in range(2))
    a, b = torch.zeros(n, 2048, device="cuda"), torch.zeros(n, 2048, device="cuda")
    check(cuda_lib.lfm_attention_prefill(ptr(q), 2048, ptr(k), ptr(v), ctx, 56, n, ptr(a), 2048, None), "prefill")
    check(cuda_lib.lfm_attention_window(shape_of("f32", 32, 8, 64, ctx), ptr(q), 2048, ptr(k), ptr(v), 56, n, 0, 0,
                                        ptr(b), 2048, None, None), "window")
    # each is within 2e-5 of the 64-bit value by its own test's bound
    assert (a - b).abs().max().item() <= 4e-5


# ------------------------------------------------------------ decode, shared
DECODE = [  # kind, heads, kv, d, ctx, lens, window, sinks, acc, pad
    ("f32", 32, 8, 64, 256, [1], 0, 0, True, 0),
    ("f32", 32, 8, 64, 700, [577, 0, 1, 31, 32, 33, 700], 0, 0, True, 512),
    ("f32", 8, 8, 128, 300, [300, 16, 17, 15], 16, 3, True, 0),
    ("f32", 6, 1, 64, 4200, [4200, 0, 4097], 1000, 40, True, 0),
    ("f16", 48, 8, 128, 513, [513, 512, 2, 100], 0, 0, True, 8),
    ("f16", 5, 1, 64, 130, [130, 64, 128, 129], 1, 0, False, 0),
    ("f16", 16, 8, 64, 2100, [2100], 2099, 0, True, 0),
    ("bf16", 32, 4, 128, 1100, [1100, 3, 0, 999], 128, 5, True, 0),
    ("bf16", 7, 7, 64, 90, [90, 89, 5], 50, 60, False, 8),
    ("bf16", 8, 1, 128, 9000, [9000], 0, 0, True, 0),
    ("f16", 8, 1, 64, 60000, [60000, 0, 53], 0, 0, True, 0),
    ("f32", 16, 8, 64, 70, [i * 70 // 63 for i in range(64)], 40, 3, False, 0),  # more CTAs than fit three to an SM
    ("bf16", 8, 4, 128, 70, [70 - i * 70 // 129 for i in range(130)], 0, 0, False, 8),
]


def decode_reference(kind, q, k, v, slots, lens, heads, kv, d, window, sinks, scale, pk=None, pv=None):
    batch = len(lens)
    out, tol = np.zeros((batch, heads * d)), np.zeros((batch, heads * d))
    acc, tol_acc = np.zeros((k.shape[0], kv, k.shape[2])), np.zeros((k.shape[0], kv, k.shape[2]))
    for b, (slot, n) in enumerate(zip(slots, lens)):
        for h in range(heads):
            kh = h // (heads // kv)
            kk, vv = k[slot, kh, :n], v[slot, kh, :n]
            see = seen(n - 1, np.arange(n), window, sinks)
            if pk is not None:
                kk, vv = np.concatenate((pk[kh], kk)), np.concatenate((pv[kh], vv))
                see = np.ones(len(kk), bool)
            at = np.flatnonzero(see)
            if at.size == 0:
                continue
            qq = q[b, h * d:(h + 1) * d]
            o, _, w = attend(qq, kk, vv, see, scale)
            ds = score_error(kind, qq, kk[at], scale)
            out[b, h * d:(h + 1) * d] = o
            tol[b, h * d:(h + 1) * d] = out_error(kind, ds, at.size, np.abs(vv[at]).max(), o)
            if pk is None:
                acc[slot, kh, :n] += w
                tol_acc[slot, kh, :n] += w * (2 * ds * (1 + ds) + 2.0 ** -20 + (at.size + 16) * 2.0 ** -23)
    return out, tol, acc, tol_acc


def session_caches(rng, kind, n_slots, kv, ctx, d, slots, lens, gap, window=0, sinks=0):
    """Caches of n_slots slots, `gap` values between them, all NaN but what a session's query sees."""
    import torch
    _, ct = torch_types(kind)
    stride = kv * ctx * d + gap
    flat = [torch.full((n_slots * stride,), float("nan"), dtype=ct) for _ in range(2)]
    views = [f.as_strided((n_slots, kv, ctx, d), (stride, ctx * d, d, 1)) for f in flat]
    for slot, n in zip(slots, lens):
        see = torch.from_numpy(seen(n - 1, np.arange(n), window, sinks))
        for x in views:
            x[slot, :, :n][:, see] = cache(rng, (kv, int(see.sum()), d), kind)
    return flat, views, stride


@pytest.mark.parametrize("kind,heads,kv,d,ctx,lens,window,sinks,with_acc,pad", DECODE)
def test_decode(cuda_lib, kind, heads, kv, d, ctx, lens, window, sinks, with_acc, pad):
    import torch
    rng = np.random.default_rng(heads + ctx)
    batch, n_slots, width = len(lens), len(lens) + 2, heads * d
    slots = rng.permutation(n_slots)[:batch]
    q = rows(rng, batch, width, kind, width + pad, 1.5)
    flat, views, stride = session_caches(rng, kind, n_slots, kv, ctx, d, slots, lens, 16, window, sinks)
    ref, tol, acc_ref, tol_acc = decode_reference(kind, f64(q), f64(views[0]), f64(views[1]), slots, lens, heads, kv,
                                                  d, window, sinks, d ** -0.5)
    qd, kd, vd = q.cuda(), flat[0].cuda(), flat[1].cuda()
    sd, ld = torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    old = torch.rand(n_slots, kv, ctx)
    accd = old.cuda() if with_acc else None
    outs = []
    for most in (max(lens), ctx):  # the host's bound does not change the result's contract
        if with_acc:
            accd.copy_(old)
        out = torch.full((batch + 1, width + 8), float("nan"), dtype=q.dtype, device="cuda")
        check(cuda_lib.lfm_attention_decode(shape_of(kind, heads, kv, d, ctx), ptr(qd), width + pad, ptr(kd), ptr(vd),
                                            stride, n_slots, ptr(sd), ptr(ld), batch, most, window, sinks, ptr(accd),
                                            ptr(out), width + 8, None), "decode")
        assert status_of(cuda_lib) == 0
        got = f64(out.cpu())
        assert np.isnan(got[:, width:]).all() and np.isnan(got[batch]).all(), "wrote outside its rows"
        err = np.abs(got[:batch, :width] - ref)
        assert (err <= tol).all(), (err.max(), (err / np.maximum(tol, 1e-30)).max())
        outs.append(got)
        if with_acc:
            want = acc_ref + old.double().numpy()
            err = np.abs(accd.cpu().double().numpy() - want)
            assert (err <= tol_acc + 2.0 ** -23 * want).all(), err.max()
            assert (err[acc_ref == 0] == 0).all()


SHARED = [  # kind, heads, kv, d, ctx, lens, prefix, pad
    ("f32", 32, 8, 64, 64, [1], 1, 0),
    ("f32", 32, 8, 64, 150, [129, 0, 1, 150], 1000, 512),
    ("f32", 8, 8, 128, 40, [40, 0, 0, 3, 17], 129, 0),
    ("f32", 20, 4, 64, 33, [33, 32, 0], 0, 0),
    ("f16", 48, 8, 128, 100, [100, 64, 2], 513, 8),
    ("f16", 6, 1, 64, 70, [5] * 45, 128, 0),
    ("bf16", 32, 4, 128, 80, list(range(0, 80, 2)), 257, 0),
    ("bf16", 7, 7, 64, 50, [0] * 3, 5000, 8),
    ("bf16", 3, 1, 128, 20, [20, 1] * 50, 127, 0),
]


@pytest.mark.parametrize("kind,heads,kv,d,ctx,lens,prefix,pad", SHARED)
def test_shared(cuda_lib, kind, heads, kv, d, ctx, lens, prefix, pad):
    import torch
    rng = np.random.default_rng(prefix + heads)
    batch, n_slots, width, pctx = len(lens), len(lens) + 1, heads * d, prefix + 9
    slots = rng.permutation(n_slots)[:batch]
    q = rows(rng, batch, width, kind, width + pad, 1.5)
    flat, views, stride = session_caches(rng, kind, n_slots, kv, ctx, d, slots, lens, 0)
    pk, pv = cache(rng, (kv, pctx, d), kind), cache(rng, (kv, pctx, d), kind)
    pk[:, prefix:], pv[:, prefix:] = float("nan"), float("nan")
    ref, tol, _, _ = decode_reference(kind, f64(q), f64(views[0]), f64(views[1]), slots, lens, heads, kv, d, 0, 0,
                                      d ** -0.5, f64(pk)[:, :prefix], f64(pv)[:, :prefix])
    qd, kd, vd, pkd, pvd = q.cuda(), flat[0].cuda(), flat[1].cuda(), pk.cuda(), pv.cuda()
    sd, ld = torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    sh = shape_of(kind, heads, kv, d, ctx)
    need = cuda_lib.lfm_attention_shared_workspace(sh, batch, prefix)
    assert need > 0
    work = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten
    out = torch.full((batch + 1, width + 8), float("nan"), dtype=q.dtype, device="cuda")
    for _ in range(2):  # the second call finds what the first left
        check(cuda_lib.lfm_attention_shared(sh, ptr(qd), width + pad, ptr(pkd), ptr(pvd), pctx, prefix, ptr(kd),
                                            ptr(vd), stride, n_slots, ptr(sd), ptr(ld), batch, max(max(lens), 1),
                                            ptr(out), width + 8, ptr(work), need, None), "shared")
        assert status_of(cuda_lib) == 0
        got = f64(out.cpu())
        assert np.isnan(got[:, width:]).all() and np.isnan(got[batch]).all(), "wrote outside its rows"
        err = np.abs(got[:batch, :width] - ref)
        assert (err <= tol).all(), (err.max(), (err / np.maximum(tol, 1e-30)).max())
    assert bool((work[need:] == 255).all()), "wrote behind its workspace"


# -------------------------------------------------------------------- evict
def evict_reference(acc, n, budget, first, last):
    """The positions one head keeps."""
    if n <= budget:
        return np.arange(n)
    lo, hi = first, n - last
    key = acc[lo:hi].astype(np.float64)
    key = np.where(np.isnan(key), -np.inf, key)
    tie = np.where(np.isnan(acc[lo:hi]), 1, 0)  # below even -inf
    order = np.lexsort((np.arange(hi - lo), tie, -key))
    middle = np.sort(order[:budget - first - last]) + lo
    return np.concatenate((np.arange(lo), middle, np.arange(hi, n)))


EVICT = [  # kv, d, ctx, lens, budget, first, last, ties
    (8, 64, 64, [64], 16, 4, 4, False),
    (2, 128, 300, [300, 299, 257, 1, 0, 100], 100, 4, 30, False),
    (3, 64, 700, [700, 512, 513, 256], 255, 0, 0, True),
    (1, 64, 5000, [5000, 4096], 2047, 33, 1000, True),
    (4, 128, 1100, [1100], 1099, 0, 1, False),
    (4, 64, 520, [520, 3], 1, 0, 0, True),
    (2, 64, 400, [400, 399], 64, 40, 24, False),
    (2, 128, 130, [130, 90], 500, 4, 4, False),
    (1, 128, 20000, [20000, 18000], 9001, 4, 64, False),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kv,d,ctx,lens,budget,first,last,ties", EVICT)
def test_evict(cuda_lib, kv, d, ctx, lens, budget, first, last, ties, in_place):
    import torch
    rng = np.random.default_rng(ctx + budget)
    batch, n_slots = len(lens), len(lens) + 1
    slots = rng.permutation(n_slots)[:batch]
    stride = kv * ctx * d + 8
    k, v = (torch.from_numpy(rng.integers(-32768, 32767, n_slots * stride, dtype=np.int16)) for _ in range(2))
    acc = rng.integers(0, 4, (n_slots, kv, ctx)).astype(np.float32) if ties else \
        np.exp(rng.normal(0, 3, (n_slots, kv, ctx))).astype(np.float32)
    acc[rng.random(acc.shape) < 0.02] = np.nan
    acc[rng.random(acc.shape) < 0.02] = -np.inf
    acc[rng.random(acc.shape) < 0.02] = np.inf
    acc[rng.random(acc.shape) < 0.05] = -0.0
    pos = rng.integers(0, 1 << 30, acc.shape).astype(np.int32)
    src = [k, v, torch.from_numpy(acc), torch.from_numpy(pos)]
    blank = [torch.full_like(x, 7) for x in src]
    want = [x.clone() for x in (src if in_place else blank)]
    for slot, n in zip(slots, lens):
        for h in range(kv):
            keep = evict_reference(acc[slot, h], n, budget, first, last)
            at = slot * stride + h * ctx * d
            for x, w in zip(src[:2], want[:2]):
                w[at:at + len(keep) * d] = x[at:at + ctx * d].view(ctx, d)[torch.from_numpy(keep)].reshape(-1)
            for x, w in zip(src[2:], want[2:]):
                w[slot, h, :len(keep)] = x[slot, h, torch.from_numpy(keep)]
    s = [x.cuda() for x in src]
    o = s if in_place else [x.cuda() for x in blank]
    sd, ld = torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    lo = torch.full((batch + 1,), -5, dtype=torch.int32, device="cuda")
    check(cuda_lib.lfm_cache_evict(shape_of("f16", kv, kv, d, ctx), *map(ptr, s), *map(ptr, o), stride, n_slots,
                                   ptr(sd), ptr(ld), ptr(lo), batch, max(lens), budget, first, last, None), "evict")
    assert status_of(cuda_lib) == 0
    assert lo.cpu().tolist() == [min(n, budget) for n in lens] + [-5]
    for i, (x, w) in enumerate(zip(o, want)):
        x = x.cpu()
        same = torch.equal(x.view(torch.int32), w.view(torch.int32)) if i >= 2 else torch.equal(x, w)
        assert same, (i, (x != w).nonzero()[:4].tolist())


# ------------------------------------------------ bad sessions, streams, runs
def test_bad_sessions_are_left_out_and_reported(cuda_lib):
    import torch
    rng = np.random.default_rng(1)
    kv, d, ctx, heads, n_slots = 2, 64, 96, 8, 3
    lens, slots = [40, 97, -1, 40, 40], [1, 0, 0, 3, -7]
    q = rows(rng, 5, heads * d, "f32", heads * d)
    k, v = cache(rng, (n_slots, kv, ctx, d), "f32"), cache(rng, (n_slots, kv, ctx, d), "f32")
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    sd, ld = torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    acc = torch.zeros(n_slots, kv, ctx, device="cuda")
    out = torch.full((5, heads * d), 3.0, device="cuda")
    sh = shape_of("f32", heads, kv, d, ctx)
    assert status_of(cuda_lib) == 0
    check(cuda_lib.lfm_attention_decode(sh, ptr(qd), heads * d, ptr(kd), ptr(vd), kv * ctx * d, n_slots, ptr(sd),
                                        ptr(ld), 5, ctx, 0, 0, ptr(acc), ptr(out), heads * d, None), "decode")
    assert status_of(cuda_lib) == 2 + 4
    assert status_of(cuda_lib) == 0
    assert bool((out[1:] == 0).all()) and bool((out[0] != 0).any())
    assert abs(acc.sum().item() - heads) < 1e-3 and abs(acc[1].sum().item() - heads) < 1e-3
    # an eviction leaves the second session of a slot out too
    slots = [1, 1, 0, 5, 2]
    lens = [40, 30, 97, 20, 96]
    sd, ld = torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    lo = torch.full((5,), -5, dtype=torch.int32, device="cuda")
    accd = torch.rand(n_slots, kv, ctx, device="cuda")
    before = kd.clone()
    check(cuda_lib.lfm_cache_evict(sh, ptr(kd), ptr(vd), ptr(accd), None, ptr(kd), ptr(vd), ptr(accd), None,
                                   kv * ctx * d, n_slots, ptr(sd), ptr(ld), ptr(lo), 5, ctx, 10, 1, 2, None), "evict")
    assert status_of(cuda_lib) == 2 + 4
    assert lo.cpu().tolist() == [10, -5, -5, -5, 10]
    assert torch.equal(kd[0], before[0])
    assert torch.equal(kd[1, :, 8:10], before[1, :, 38:40])


def test_serving_steps_together(cuda_lib):
    """Prompt, weights, decode steps with accumulated weights and an eviction in place, captured once as a graph
    and replayed on another stream, against the same steps in 64 bits."""
    import torch
    rng = np.random.default_rng(9)
    heads, kv, d, ctx, n, budget, first, last = 8, 2, 64, 160, 120, 64, 4, 16
    w, g = heads * d, heads // kv
    q = rows(rng, n, w, "f32", w, 1.5)
    qs = rows(rng, 2, w, "f32", w, 1.5)
    k, v = cache(rng, (2, kv, ctx, d), "f32"), cache(rng, (2, kv, ctx, d), "f32")
    sh = shape_of("f32", heads, kv, d, ctx)
    qd, qsd = q.cuda(), qs.cuda()
    kd, vd = k.cuda(), v.cuda()
    acc = torch.zeros(2, kv, ctx, device="cuda")
    pos = torch.arange(ctx, dtype=torch.int32).expand(2, kv, ctx).contiguous().cuda()
    out, o1, o2 = (torch.zeros(m, w, device="cuda") for m in (n, 2, 2))
    lse = torch.zeros(n, heads, device="cuda")
    ld = torch.tensor([n, n - 7], dtype=torch.int32, device="cuda")
    lo = torch.zeros(2, dtype=torch.int32, device="cuda")
    slot = kv * ctx * d
    start = [x.clone() for x in (kd, vd, acc, pos)]

    def steps(stream):
        for s in range(2):
            at = ctypes.c_void_p(kd.data_ptr() + s * slot * 2), ctypes.c_void_p(vd.data_ptr() + s * slot * 2)
            check(cuda_lib.lfm_attention_window(sh, ptr(qd), w, *at, 0, n, 50, 4, ptr(out), w, ptr(lse), stream), "w")
            check(cuda_lib.lfm_attention_weights(sh, ptr(qd), w, at[0], 0, n, 50, 4, ptr(lse),
                                                 ctypes.c_void_p(acc.data_ptr() + s * kv * ctx * 4), stream), "a")
        args = (ptr(kd), ptr(vd), slot, 2, None)
        check(cuda_lib.lfm_attention_decode(sh, ptr(qsd), w, *args, ptr(ld), 2, ctx, 0, 0, ptr(acc), ptr(o1), w,
                                            stream), "d")
        check(cuda_lib.lfm_cache_evict(sh, ptr(kd), ptr(vd), ptr(acc), ptr(pos), ptr(kd), ptr(vd), ptr(acc), ptr(pos),
                                       slot, 2, None, ptr(ld), ptr(lo), 2, ctx, budget, first, last, stream), "e")
        check(cuda_lib.lfm_attention_decode(sh, ptr(qsd), w, *args, ptr(lo), 2, budget, 0, 0, ptr(acc), ptr(o2), w,
                                            stream), "d")

    def reset():
        for x, y in zip((kd, vd, acc, pos), start):
            x.copy_(y)

    steps(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert status_of(cuda_lib) == 0
    eager = [x.clone() for x in (o1, o2, acc, pos, kd, lo)]
    # the same in 64 bits, by the positions that the kernels kept (their choice is checked against the weights)
    k64, v64 = f64(k), f64(v)
    for s, m in enumerate((n, n - 7)):
        total = np.zeros((kv, ctx))
        for t in range(n):
            see = seen(t, np.arange(t + 1), 50, 4)
            for h in range(heads):
                total[h // g, :t + 1] += attend(f64(q)[t, h * d:(h + 1) * d], k64[s, h // g, :t + 1],
                                                v64[s, h // g, :t + 1], see, d ** -0.5)[2]
        for h in range(heads):
            qq = f64(qs)[s, h * d:(h + 1) * d]
            o, _, ww = attend(qq, k64[s, h // g, :m], v64[s, h // g, :m], np.ones(m, bool), d ** -0.5)
            total[h // g, :m] += ww
            assert np.abs(o1[s, h * d:(h + 1) * d].cpu().double().numpy() - o).max() < 1e-4
        for h in range(heads):
            kept = pos[s, h // g, :budget].cpu().numpy()
            assert (np.diff(kept) > 0).all() and kept[:first].tolist() == list(range(first))
            assert kept[-last:].tolist() == list(range(m - last, m))
            t = total[h // g, first:m - last]
            lowest = np.sort(t)[::-1][budget - first - last - 1]
            assert (total[h // g, kept[first:-last]] >= lowest * (1 - 1e-4)).all()
            qq = f64(qs)[s, h * d:(h + 1) * d]
            o = attend(qq, k64[s, h // g, kept], v64[s, h // g, kept], np.ones(budget, bool), d ** -0.5)[0]
            assert np.abs(o2[s, h * d:(h + 1) * d].cpu().double().numpy() - o).max() < 1e-4
    # captured on another stream and replayed twice from the same start
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        steps(ctypes.c_void_p(side.cuda_stream))
        graph.capture_end()
    torch.cuda.synchronize()
    for _ in range(2):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((o1, o2, acc, pos, kd, lo), eager):
            assert torch.equal(x, y)
    assert status_of(cuda_lib) == 0


def _shared_state(seed, batch=24, prefix=300, heads=8, kv=2, d=64, ctx=48):
    import torch
    rng = np.random.default_rng(seed)
    sh = shape_of("bf16", heads, kv, d, ctx)
    q = rows(rng, batch, heads * d, "bf16", heads * d).cuda()
    k, v = (cache(rng, (batch, kv, ctx, d), "bf16").cuda() for _ in range(2))
    pk, pv = (cache(rng, (kv, prefix, d), "bf16").cuda() for _ in range(2))
    lens = torch.from_numpy(rng.integers(0, ctx + 1, batch).astype(np.int32)).cuda()
    return sh, q, k, v, pk, pv, lens


def _shared_call(lib, state, out, work, stream):
    sh, q, k, v, pk, pv, lens = state
    b, w = q.shape
    check(lib.lfm_attention_shared(sh, ptr(q), w, ptr(pk), ptr(pv), pk.shape[1], pk.shape[1], ptr(k), ptr(v),
                                   k.stride(0), b, None, ptr(lens), b, sh.ctx, ptr(out), w, ptr(work), work.numel(),
                                   ctypes.c_void_p(stream.cuda_stream)), "shared")


def test_shared_captured_replayed_and_on_two_streams(cuda_lib):
    """The call's two kernels in a graph that is replayed after its inputs have changed, and two calls at once on two
    streams with a workspace each."""
    import torch
    a, b = _shared_state(1), _shared_state(2)
    need = cuda_lib.lfm_attention_shared_workspace(a[0], 24, 300)
    work = [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want, main = [], torch.cuda.current_stream()
    for s in (a, b):
        out = torch.zeros_like(s[1])
        _shared_call(cuda_lib, s, out, work[0], main)
        want.append(out)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(want[0]) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w, t in zip((a, b), outs, work, side):
            _shared_call(cuda_lib, s, o, w, t)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    out = torch.zeros_like(want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side[0]):
        graph.capture_begin()
        _shared_call(cuda_lib, a, out, work[0], side[0])
        graph.capture_end()
    for x, y in zip(a[1:], b[1:]):
        x.copy_(y)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[1])
    assert status_of(cuda_lib) == 0


def test_first_call_of_a_process_inside_a_capture():
    """No call needs one before it: the kernels' attributes and maps are set while the stream captures."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch, ctypes, conftest, lfm2_b200
from test_gpu_cache_attn import _shared_state, _shared_call
lib = lfm2_b200.lib()
s = _shared_state(3)
work = torch.zeros(lib.lfm_attention_shared_workspace(s[0], 24, 300), dtype=torch.uint8, device="cuda")
out, again = torch.zeros_like(s[1]), torch.zeros_like(s[1])
torch.cuda.synchronize()
side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.stream(side):
    g.capture_begin()
    _shared_call(lib, s, out, work, side)
    g.capture_end()
g.replay()
torch.cuda.synchronize()
_shared_call(lib, s, again, work, torch.cuda.current_stream())
torch.cuda.synchronize()
assert torch.equal(out, again) and bool((out != 0).any())
print("same")
""" % (here, os.path.join(os.path.dirname(here), "lfm2-w9100-rust_b200"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_offsets_past_32_bits(cuda_lib):
    """A session whose cache starts 4.7e9 values into the array, its positions evicted in place there."""
    import torch
    kv, d, ctx, heads, slot = 8, 64, 1 << 17, 8, 70
    stride = kv * ctx * d
    k = torch.zeros((slot + 1) * stride, dtype=torch.float16, device="cuda")
    v = torch.zeros((slot + 1) * stride, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(4)
    n = 200
    q = rows(rng, 1, heads * d, "f16", heads * d)
    kk, vv = cache(rng, (kv, n, d), "f16"), cache(rng, (kv, n, d), "f16")
    at = slot * stride
    kview, vview = k[at:].view(kv, ctx, d), v[at:].view(kv, ctx, d)
    kview[:, :n], vview[:, :n] = kk.cuda(), vv.cuda()
    sh = shape_of("f16", heads, kv, d, ctx)
    sd, ld = torch.tensor([slot], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    acc = torch.zeros(slot + 1, kv, ctx, device="cuda")
    out = torch.zeros(1, heads * d, dtype=torch.float16, device="cuda")
    qd, lo = q.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    check(cuda_lib.lfm_attention_decode(sh, ptr(qd), heads * d, ptr(k), ptr(v), stride, slot + 1, ptr(sd), ptr(ld), 1,
                                        ctx, 0, 0, ptr(acc), ptr(out), heads * d, None), "decode")
    for h in range(heads):
        o, _, w = attend(f64(q)[0, h * d:(h + 1) * d], f64(kk)[h], f64(vv)[h], np.ones(n, bool), d ** -0.5)
        ds = score_error("f16", f64(q)[0, h * d:(h + 1) * d], f64(kk)[h], d ** -0.5)
        tol = out_error("f16", ds, n, np.abs(f64(vv)[h]).max(), o)
        assert (np.abs(out[0, h * d:(h + 1) * d].cpu().double().numpy() - o) <= tol).all()
        assert np.abs(acc[slot, h, :n].cpu().double().numpy() - w).max() < 1e-5
    assert acc[:slot].abs().max().item() == 0
    check(cuda_lib.lfm_cache_evict(sh, ptr(k), ptr(v), ptr(acc), None, ptr(k), ptr(v), ptr(acc), None, stride, slot + 1,
                                   ptr(sd), ptr(ld), ptr(lo), 1, n, 50, 0, 50, None), "evict")
    assert torch.equal(kview[:, :50], kk[:, 150:].cuda()) and torch.equal(vview[:, :50], vv[:, 150:].cuda())
    assert status_of(cuda_lib) == 0


def test_memory_of_the_host_is_refused(cuda_lib):
    import torch
    x = torch.zeros(1 << 16)
    y = torch.zeros(1 << 16, device="cuda")
    sh = shape_of("f32", 8, 2, 64, 64)
    assert cuda_lib.lfm_attention_window(sh, ptr(x), 512, ptr(y), ptr(y), 0, 4, 0, 0, ptr(y), 512, None, None) == 1
    assert cuda_lib.lfm_attention_window(sh, ptr(y), 512, ptr(y), ptr(x), 0, 4, 0, 0, ptr(y), 512, None, None) == 1
    assert cuda_lib.lfm_attention_weights(sh, ptr(y), 512, ptr(y), 0, 4, 0, 0, ptr(x), ptr(y), None) == 1
    assert cuda_lib.lfm_attention_decode(sh, ptr(y), 512, ptr(y), ptr(y), 8192, 1, None, ptr(x), 1, 64, 0, 0, None,
                                         ptr(y), 512, None) == 1
    assert b"current device" in cuda_lib.lfm_ops_error()
