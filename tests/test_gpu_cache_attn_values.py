"""Values that are not finite in the session-cache attention calls."""

import pytest

from cache_attn_ref import torch_types
from test_gpu_cache_attn import status_of
from test_gpu_cache_attn_precision import decode, shared, window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,d", [("f32", 64), ("f32", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("first,end", [(0, 2048), (1000, 1001), (2560, 4096), (4095, 4096), (0, 4096)])
def test_nan_keys_reach_every_query_that_sees_them(cuda_lib, kind, d, first, end):
    """Also where all that one CTA of a split row, or one warp, sees is NaN: its part has no maximum."""
    import torch
    heads, kv, n = 4, 1, 4096
    g = torch.Generator(device="cuda").manual_seed(first + end)
    qt, ct = torch_types(kind)
    q = torch.randn(1, heads * d, generator=g, device="cuda").to(qt)
    k, v = (torch.randn(kv, n, d, generator=g, device="cuda").to(ct) for _ in range(2))
    empty = k[None, :, :1].contiguous(), v[None, :, :1].contiguous()

    def outs():
        return (window(cuda_lib, kind, heads, q, k, v, n - 1), decode(cuda_lib, kind, heads, q, k[None], v[None], [n]),
                shared(cuda_lib, kind, heads, q, k, v, *empty, [0]),
                shared(cuda_lib, kind, heads, q, k[:, :2048].contiguous(), v[:, :2048].contiguous(),
                       k[None, :, 2048:].contiguous(), v[None, :, 2048:].contiguous(), [2048]))

    assert all(bool(torch.isfinite(o).all()) for o in outs())
    k[:, first:end] = float("nan")
    for i, o in enumerate(outs()):
        assert bool(torch.isnan(o).all()), i
    assert status_of(cuda_lib) == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size,scale", [(0.0, 0.0), (0.0, 2.0 ** -100), (2.0 ** -120, 2.0 ** -100), (2.0 ** -120, 2.0 ** 100)])
def test_queries_and_scales_at_the_ends_of_fp32(cuda_lib, d, size, scale):
    """Scores so small that every seen position weighs the same, under a causal mask and a window: means of V."""
    import torch
    from cache_attn_ref import ptr
    from test_gpu_cache_attn import check, shape_of
    heads, kv, n, window_, sinks = 4, 1, 300, 100, 3
    g = torch.Generator(device="cuda").manual_seed(d)
    q = size * torch.randn(n, heads * d, generator=g, device="cuda")
    k, v = (torch.randn(kv, n, d, generator=g, device="cuda").half() for _ in range(2))
    out, lse = torch.full_like(q, float("nan")), torch.zeros(n, heads, device="cuda")
    sh = shape_of("f32", heads, kv, d, n, scale)
    check(cuda_lib.lfm_attention_window(sh, ptr(q), heads * d, ptr(k), ptr(v), 0, n, window_, sinks, ptr(out), heads * d,
                                        ptr(lse), None), "window")
    acc = torch.zeros(kv, n, device="cuda")
    check(cuda_lib.lfm_attention_weights(sh, ptr(q), heads * d, ptr(k), 0, n, window_, sinks, ptr(lse), ptr(acc), None), "w")
    last = torch.full((1, heads * d), float("nan"), device="cuda")
    ld = torch.tensor([n], dtype=torch.int32, device="cuda")
    check(cuda_lib.lfm_attention_decode(sh, ptr(q[-1]), heads * d, ptr(k), ptr(v), kv * n * d, 1, None, ptr(ld), 1, n,
                                        window_, sinks, None, ptr(last), heads * d, None), "decode")
    assert status_of(cuda_lib) == 0
    p, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    see = ((j <= p) & ((p - j < window_) | (j < sinks))).double()
    w = see / see.sum(1, keepdim=True)
    mean = w @ v[0].double()
    # equal weights of fp32 pairs, sums of at most 103 of them and of their products: 2^-22 + 2 * 103 * 2^-23 of max |v|
    most = (2.0 ** -22 + 206 * 2.0 ** -23) * v.abs().max().item()
    got = out.double().view(n, heads, d)
    assert (got - mean[:, None]).abs().max().item() <= most
    assert (last.double().view(heads, d) - mean[-1]).abs().max().item() <= most
    assert (acc[0].double() - heads * w.sum(0)).abs().max().item() <= 1200 * 2.0 ** -23 * heads * w.sum(0).max().item()
