"""Values that are not finite in the session-cache attention calls."""

import pytest

from cache_attn_ref import torch_types
from test_gpu_cache_attn import status_of
from test_gpu_cache_attn_precision import decode, shared, window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,d", [("f32", 64), ("f32", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("first,end", [(0, 2048), (1000, 1001), (3072, 4096), (4095, 4096), (0, 4096)])
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
