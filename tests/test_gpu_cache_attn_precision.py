"""Precision of the session-cache attention calls against 64-bit values, in
norm and on the inputs where a number format shows (limits: cache_attn_norm)."""

import numpy as np
import pytest

from cache_attn_norm import SHIFT, dominated, fp16_floor, limit, norm_error, plain32, score_cut
from cache_attn_ref import attend, ptr, seen, torch_types
from test_gpu_cache_attn import check, f64, shape_of, status_of

pytestmark = pytest.mark.gpu


def on_gpu(x, kind, cache):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch_types(kind)[1 if cache else 0]).cuda()


def decode(lib, kind, heads, q, k, v, lens, acc=None):
    """q [batch][heads * d], k and v [batch][kv][ctx][d]."""
    import torch
    batch, kv, ctx, d = k.shape
    out = torch.full_like(q, float("nan"))
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check(lib.lfm_attention_decode(shape_of(kind, heads, kv, d, ctx), ptr(q), heads * d, ptr(k), ptr(v), kv * ctx * d,
                                   batch, None, ptr(ld), batch, max(lens), 0, 0, ptr(acc), ptr(out), heads * d, None),
          "decode")
    return out


def window(lib, kind, heads, q, k, v, start, lse=None):
    """q [n][heads * d], k and v [kv][ctx][d]."""
    import torch
    kv, ctx, d = k.shape
    out = torch.full_like(q, float("nan"))
    check(lib.lfm_attention_window(shape_of(kind, heads, kv, d, ctx), ptr(q), heads * d, ptr(k), ptr(v), start, len(q),
                                   0, 0, ptr(out), heads * d, ptr(lse), None), "window")
    return out


def shared(lib, kind, heads, q, pk, pv, k, v, lens):
    """q [batch][heads * d], pk and pv [kv][prefix][d], k and v [batch][kv][ctx][d]."""
    import torch
    batch, kv, ctx, d = k.shape
    prefix = pk.shape[1]
    sh = shape_of(kind, heads, kv, d, ctx)
    out = torch.full_like(q, float("nan"))
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    need = lib.lfm_attention_shared_workspace(sh, batch, prefix)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    check(lib.lfm_attention_shared(sh, ptr(q), heads * d, ptr(pk), ptr(pv), prefix, prefix, ptr(k), ptr(v), kv * ctx * d,
                                   batch, None, ptr(ld), batch, max(max(lens), 1), ptr(out), heads * d, ptr(work), need,
                                   None), "shared")
    return out


def row_errors(kind, q, k, v, got, growth=0.0, see=None):
    """The error in norm and its limit for rows got [heads][d] over k, v [kv][n][d]; `growth` is the power of two that
    the kernel leaves free above the largest weight (fp16 queries of many rows: 2^8)."""
    heads, d = q.shape
    g, every = heads // len(k), np.ones(k.shape[1], bool) if see is None else see
    k, v, every = k[:, every], v[:, every], every[every]
    rows = [attend(q[h], k[h // g], v[h // g], every, d ** -0.5) for h in range(heads)]
    want = np.stack([r[0] for r in rows])
    floor = np.linalg.norm([fp16_floor(r[2], v[h // g], SHIFT[kind] - growth) for h, r in enumerate(rows)])
    floor = 0.0 if kind == "bf16" else floor / np.linalg.norm(want)
    floor += max(score_cut(d, k[h // g] @ q[h] * d ** -0.5) for h in range(heads))
    plain = np.stack([plain32(q[h], k[h // g], v[h // g], d ** -0.5) for h in range(heads)])
    return norm_error(got, want), limit(kind, norm_error(plain, want), floor)


@pytest.mark.parametrize("kind,d,nats", [(kind, d, nats) for kind in ("f32", "f16", "bf16") for d in (64, 128)
                                         for nats in (6, 10) + ((14,) if kind != "f16" else ())])
def test_a_key_that_takes_the_weight_over_a_zero_value(cuda_lib, kind, d, nats):
    """A sink's place: one key far above the others, its value row 0. The error is relative to what is left."""
    heads, kv, n, at = 8, 2, 3000, 3
    q, k, v = dominated(np.random.default_rng(d + nats), kind, heads, kv, n, d, nats, at)
    qd, kd, vd = on_gpu(q.reshape(1, -1), kind, False), on_gpu(k, kind, True), on_gpu(v, kind, True)
    empty = kd[None, :, :1].contiguous(), vd[None, :, :1].contiguous()
    outs = {"decode": decode(cuda_lib, kind, heads, qd, kd[None], vd[None], [n]),
            "window": window(cuda_lib, kind, heads, qd, kd, vd, n - 1),
            "shared": shared(cuda_lib, kind, heads, qd, kd, vd, *empty, [0]),
            "joined": shared(cuda_lib, kind, heads, qd, kd[:, :1000].contiguous(), vd[:, :1000].contiguous(),
                             kd[None, :, 1000:].contiguous(), vd[None, :, 1000:].contiguous(), [n - 1000])}
    assert status_of(cuda_lib) == 0
    for name, out in outs.items():
        error, most = row_errors(kind, q, k, v, f64(out.cpu()).reshape(heads, d),
                                 8.0 if kind == "f16" and name != "decode" else 0.0)
        assert error <= most, (name, error, most)


def long_rows(seed, kind, heads, kv, n, d, batch):
    """Queries, and keys and values of n positions that every session shares, the values positive: an error that grows
    with the number of positions adds up instead of averaging out."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    qt, ct = torch_types(kind)
    q = torch.randn(batch, heads * d, generator=g, device="cuda").to(qt)
    k = torch.randn(kv, n, d, generator=g, device="cuda").to(ct)
    v = (torch.rand(kv, n, d, generator=g, device="cuda") + 0.5).to(ct)
    return q, k, v


def long_reference(q, k, v, heads):
    """64-bit outputs [batch][heads][d]."""
    import torch
    kv, _, d = k.shape
    x = q.double().view(-1, kv, heads // kv, d) * d ** -0.5
    out = torch.stack([torch.softmax(x[:, h] @ k[h].double().T, -1) @ v[h].double() for h in range(kv)], 1)
    return out.reshape(-1, heads, d)


def mean_error(out, want):
    """Relative to the 64-bit value, of the distance from that value rounded to the output's type: near a power of two,
    which the outputs straddle, the steps above are twice those below, so that rounding alone has a mean that is not 0
    (outputs of mean 1 and deviation s: -(2^-23 - 2^-25) / (s sqrt(2 pi)) in fp16)."""
    return ((out.double().view_as(want) - want.to(out.dtype).double()) / want).mean().item()


# What a long sum may lose in the mean of all outputs. fp32 queries: a tile or chunk of up to eight sums cut off by less
# than 2^-23 each. fp16: the same up to a fold, 256 sums on the way up to the value, half a step of 2^-23 lost in the mean
# of each, and six standard deviations of the mean of `count` roundings to fp16 (uniform in half a step of 2^-11).
def most_bias(kind, count):
    return 8 * 2.0 ** -23 if kind == "f32" else 256 * 2.0 ** -25 + 6 * 2.0 ** -11 / np.sqrt(3 * count)


@pytest.mark.parametrize("kind,heads,kv,n,d,batch", [("f32", 8, 2, 16385, 64, 80), ("f32", 8, 1, 200001, 128, 1),
                                                     ("f32", 4, 1, 1 << 20, 64, 1), ("f16", 8, 1, 1 << 20, 64, 1)])
def test_long_sums_of_one_token(cuda_lib, kind, heads, kv, n, d, batch):
    q, k, v = long_rows(n, kind, heads, kv, n, d, batch)
    every = [x[None].expand(batch, kv, n, d).contiguous() for x in (k, v)]
    out = decode(cuda_lib, kind, heads, q, *every, [n] * batch)
    want = long_reference(q, k, v, heads)
    bias = mean_error(out, want)
    assert status_of(cuda_lib) == 0
    assert abs(bias) <= most_bias(kind, want.numel()), bias


@pytest.mark.parametrize("kind,heads,kv,n,d", [("f32", 8, 1, 1 << 18, 64), ("f16", 8, 1, 1 << 20, 64),
                                               ("f16", 8, 1, 1 << 20, 128)])
def test_long_sums_of_many_rows(cuda_lib, kind, heads, kv, n, d):
    """The prompt's last rows and the rows behind a shared prefix, over so many tiles that each CTA folds."""
    q, k, v = long_rows(n, kind, heads, kv, n, d, 3)
    want = long_reference(q, k, v, heads)
    empty = [x[None, :, :1].expand(3, kv, 1, d).contiguous() for x in (k, v)]
    out = shared(cuda_lib, kind, heads, q, k, v, *empty, [0, 0, 0])
    bias = mean_error(out, want)
    assert abs(bias) <= most_bias(kind, want.numel()), bias
    out = window(cuda_lib, kind, heads, q, k, v, n - 3)[2]  # of the three rows, the one that sees all
    bias = mean_error(out, want[2])
    assert abs(bias) <= most_bias(kind, want[2].numel()), bias
    assert status_of(cuda_lib) == 0


@pytest.mark.parametrize("kind,d", [("f16", 64), ("bf16", 128)])
def test_a_maximum_that_rises_across_folds(cuda_lib, kind, d):
    """Scores that grow along the positions: outputs folded early are relative to maxima that later ones outgrow, by
    little (the maximum is not raised) and by much."""
    import torch
    heads, kv, n = 4, 1, 70000
    g = torch.Generator(device="cuda").manual_seed(d)
    qt, ct = torch_types(kind)
    q = torch.randn(1, heads * d, generator=g, device="cuda").to(qt)
    for rise in (3.0, 40.0):
        x = q.double().view(heads, d)[0]
        k = 0.3 * torch.randn(kv, n, d, generator=g, device="cuda", dtype=torch.float64)
        k[0] += torch.linspace(0, rise, n, device="cuda", dtype=torch.float64)[:, None] * x * d ** 0.5 / (x @ x)
        k, v = k.to(ct), torch.randn(kv, n, d, generator=g, device="cuda").to(ct)
        out = window(cuda_lib, kind, heads, q, k, v, n - 1)
        assert status_of(cuda_lib) == 0
        for h in range(heads):
            error, most = row_errors(kind, f64(q.cpu()).reshape(heads, d)[h:h + 1], f64(k.cpu()), f64(v.cpu()),
                                     f64(out.cpu()).reshape(heads, d)[h:h + 1], 8.0)
            assert error <= most, (rise, h, error, most)


@pytest.mark.parametrize("d", [64, 128])
def test_fp32_queries_of_any_size(cuda_lib, d):
    """Rows of one call whose queries differ by many orders of magnitude, against keys of the inverse size: fp32 holds
    them all alike. One KV head to a size."""
    import torch
    sizes = [1e-4, 1e-2, 1.0, 40.0, 3e5]
    kv, n, g = len(sizes), 400, 2
    heads, rng = g * kv, np.random.default_rng(d)
    x = (rng.normal(0, 1, (heads, d)) * np.repeat(sizes, g)[:, None]).astype(np.float32)
    k = (rng.normal(0, 1, (kv, n, d)) / np.array(sizes)[:, None, None]).astype(np.float16)
    v = rng.normal(0, 1, (kv, n, d)).astype(np.float16)
    assert np.isfinite(k).all()
    x, k, v = x.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    qd, kd, vd = on_gpu(x.reshape(1, -1), "f32", False), on_gpu(k, "f32", True), on_gpu(v, "f32", True)
    empty = kd[None, :, :1].contiguous(), vd[None, :, :1].contiguous()
    acc, lse = torch.zeros(1, kv, n, device="cuda"), torch.zeros(1, heads, device="cuda")
    outs = {"decode": decode(cuda_lib, "f32", heads, qd, kd[None], vd[None], [n], acc),
            "window": window(cuda_lib, "f32", heads, qd, kd, vd, n - 1, lse),
            "shared": shared(cuda_lib, "f32", heads, qd, kd, vd, *empty, [0])}
    for name, out in outs.items():
        got = f64(out.cpu()).reshape(heads, d)
        for h in range(kv):
            rows = slice(h * g, (h + 1) * g)
            error, most = row_errors("f32", x[rows], k[h:h + 1], v[h:h + 1], got[rows])
            assert error <= most, (name, sizes[h], error, most)
    acc2 = torch.zeros(kv, n, device="cuda")
    check(cuda_lib.lfm_attention_weights(shape_of("f32", heads, kv, d, n), ptr(qd), heads * d, ptr(kd), n - 1, 1, 0, 0,
                                         ptr(lse), ptr(acc2), None), "weights")
    assert status_of(cuda_lib) == 0
    for h in range(kv):
        s = x[h * g:(h + 1) * g] @ k[h].T * d ** -0.5
        w = np.exp(s - s.max(1, keepdims=True))
        want = (w / w.sum(1, keepdims=True)).sum(0)
        s32 = (x[h * g:(h + 1) * g].astype(np.float32) @ k[h].T.astype(np.float32)) * np.float32(d ** -0.5)
        w32 = np.exp(s32 - s32.max(1, keepdims=True))
        plain = norm_error((w32 / w32.sum(1, keepdims=True)).sum(0), want)
        most = limit("f32", plain, score_cut(d, s))
        for got in (acc[0, h], acc2[h]):
            assert norm_error(f64(got.cpu()), want) <= most, (sizes[h], norm_error(f64(got.cpu()), want), most)


@pytest.mark.parametrize("kind,start,n,window_,sinks", [("f32", 300, 40, 50, 4), ("bf16", 129, 1, 1, 0),
                                                        ("f16", 512, 128, 128, 131)])
def test_weights_leave_the_records_that_no_query_sees(cuda_lib, kind, start, n, window_, sinks):
    """Positions between the sinks and the first window, and behind the last query: not a bit changes (-0 stays -0)."""
    import torch
    heads, kv, d, ctx = 8, 2, 64, start + n + 70
    g = torch.Generator(device="cuda").manual_seed(start)
    qt, ct = torch_types(kind)
    q = torch.randn(n, heads * d, generator=g, device="cuda").to(qt)
    k, v = (torch.randn(kv, ctx, d, generator=g, device="cuda").to(ct) for _ in range(2))
    lse = torch.zeros(n, heads, device="cuda")
    sh = shape_of(kind, heads, kv, d, ctx)
    check(cuda_lib.lfm_attention_window(sh, ptr(q), heads * d, ptr(k), ptr(v), start, n, window_, sinks,
                                        ptr(torch.empty_like(q)), heads * d, ptr(lse), None), "window")
    acc = torch.full((kv, ctx), -0.0, device="cuda")
    check(cuda_lib.lfm_attention_weights(sh, ptr(q), heads * d, ptr(k), start, n, window_, sinks, ptr(lse), ptr(acc), None),
          "weights")
    assert status_of(cuda_lib) == 0
    j = np.arange(ctx)
    hidden = (j >= start + n) | ((j >= sinks) & (j <= start - window_))
    got = acc.cpu().numpy()
    assert (got.view(np.uint32)[:, hidden] == 0x80000000).all() and hidden.sum() > 70
    assert (got[:, ~hidden] > 0).all()


# The shapes of the calls in earnest, each row against the limit of its own type; a call's fp32 path that loses a half of
# its pairs is off by 2e-4 where 2e-6 to 4e-6 are allowed.
NORM = [  # kind, heads, kv, d, lens, window, sinks, prefix
    ("f32", 32, 8, 64, [577, 1, 33, 2000], 0, 0, 500),
    ("f32", 16, 8, 128, [300, 17, 128], 0, 0, 129),
    ("f32", 6, 1, 64, [3000, 40], 1000, 40, 1),
    ("f32", 8, 1, 128, [5000], 128, 5, 2000),
    ("f16", 32, 8, 64, [577, 1, 33], 0, 0, 500),
    ("f16", 12, 2, 128, [3000, 63], 700, 3, 64),
    ("bf16", 32, 4, 128, [1100, 3, 999], 128, 5, 300),
    ("bf16", 7, 7, 64, [90, 2048], 0, 0, 1000),
]


@pytest.mark.parametrize("kind,heads,kv,d,lens,window_,sinks,prefix", NORM)
def test_errors_in_norm(cuda_lib, kind, heads, kv, d, lens, window_, sinks, prefix):
    import torch
    batch, ctx = len(lens), max(lens) + 5
    g = torch.Generator(device="cuda").manual_seed(heads * d)
    qt, ct = torch_types(kind)
    q = (1.5 * torch.randn(batch, heads * d, generator=g, device="cuda")).to(qt)
    k, v = (torch.randn(batch, kv, ctx, d, generator=g, device="cuda").to(ct) for _ in range(2))
    pk, pv = (torch.randn(kv, prefix, d, generator=g, device="cuda").to(ct) for _ in range(2))
    sh, ld = shape_of(kind, heads, kv, d, ctx), torch.tensor(lens, dtype=torch.int32, device="cuda")
    stepped, acc = torch.empty_like(q), torch.zeros(batch, kv, ctx, device="cuda")
    check(cuda_lib.lfm_attention_decode(sh, ptr(q), heads * d, ptr(k), ptr(v), kv * ctx * d, batch, None, ptr(ld), batch,
                                        max(lens), window_, sinks, ptr(acc), ptr(stepped), heads * d, None), "decode")
    behind = shared(cuda_lib, kind, heads, q, pk, pv, k, v, lens)
    prompt = torch.empty_like(q)
    for b, n in enumerate(lens):  # each session's newest token as a prompt of one
        check(cuda_lib.lfm_attention_window(sh, ptr(q[b]), heads * d, ptr(k[b]), ptr(v[b]), n - 1, 1, window_, sinks,
                                            ptr(prompt[b]), heads * d, None, None), "window")
    assert status_of(cuda_lib) == 0
    q64, k64, v64, pk64, pv64 = (f64(x.cpu()) for x in (q, k, v, pk, pv))
    growth = 8.0 if kind == "f16" else 0.0
    for b, n in enumerate(lens):
        see = seen(n - 1, np.arange(n), window_, sinks)
        for out, how, least in ((stepped, see, 0.0), (prompt, see, growth), (behind, None, growth)):
            kk, vv = k64[b, :, :n], v64[b, :, :n]
            if how is None:
                kk, vv = np.concatenate((pk64, kk), 1), np.concatenate((pv64, vv), 1)
            error, most = row_errors(kind, q64[b].reshape(heads, d), kk, vv, f64(out[b].cpu()).reshape(heads, d), least, how)
            assert error <= most, (b, out is stepped, out is prompt, error, most)


@pytest.mark.parametrize("kind,d", [("f16", 64), ("bf16", 128)])
def test_many_long_rows(cuda_lib, kind, d):
    """A prompt's chunk deep in a long cache: enough rows that each CTA walks all positions of its rows and folds, with
    the causal edge, and the window's, in the tiles behind."""
    import torch
    heads, kv, n, start = 16, 2, 1200, 5000
    g = torch.Generator(device="cuda").manual_seed(d)
    qt, ct = torch_types(kind)
    q = (1.5 * torch.randn(n, heads * d, generator=g, device="cuda")).to(qt)
    k, v = (torch.randn(kv, start + n, d, generator=g, device="cuda").to(ct) for _ in range(2))
    sh = shape_of(kind, heads, kv, d, start + n)
    for window_, sinks in ((0, 0), (4700, 70)):
        out = torch.full_like(q, float("nan"))
        check(cuda_lib.lfm_attention_window(sh, ptr(q), heads * d, ptr(k), ptr(v), start, n, window_, sinks, ptr(out),
                                            heads * d, None, None), "window")
        assert status_of(cuda_lib) == 0
        p, j = torch.arange(start, start + n, device="cuda")[:, None], torch.arange(start + n, device="cuda")[None]
        see = (j <= p) & ((p - j < window_) | (j < sinks)) if window_ else j <= p
        for h in range(heads):
            x = q.view(n, heads, d)[:, h].double() @ k[h // 8].double().T * d ** -0.5
            want = torch.softmax(x.masked_fill(~see, float("-inf")), -1) @ v[h // 8].double()
            got = out.view(n, heads, d)[:, h].double()
            error = ((got - want).norm(dim=1) / want.norm(dim=1)).max().item()
            assert error <= limit(kind, 0.0, score_cut(d, x[see].abs().max().item())), (h, error)
