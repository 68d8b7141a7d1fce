"""What the session-cache attention calls refuse before they launch anything
(no GPU: the pointers are never followed), and the layout of their shape."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

A = 1 << 20  # stands for a device pointer


def _lib():
    import lfm2_b200
    return lfm2_b200, lfm2_b200.lib()


def _shape(**kw):
    m, _ = _lib()
    base = dict(dtype=0, heads=8, kv_heads=2, head_dim=64, ctx=128, scale=0.0)
    base.update(kw)
    return m.AttnShape(*[base[f] for f, _ in m.AttnShape._fields_])


BAD_SHAPES = [dict(dtype=3), dict(kv_heads=0), dict(kv_heads=1025, heads=1025), dict(head_dim=96), dict(ctx=0),
              dict(ctx=(1 << 24) + 1), dict(heads=7), dict(heads=18), dict(heads=0), dict(scale=-1.0),
              dict(scale=float("nan")), dict(scale=float("inf"))]


def window(sh=None, q=A, qs=512, k=A, v=A, start=0, n=4, w=0, s=0, out=A, os_=512, lse=None):
    return _lib()[1].lfm_attention_window(sh or _shape(), q, qs, k, v, start, n, w, s, out, os_, lse, None)


def weights(sh=None, q=A, qs=512, k=A, start=0, n=4, lse=A, acc=A):
    return _lib()[1].lfm_attention_weights(sh or _shape(), q, qs, k, start, n, 0, 0, lse, acc, None)


def decode(sh=None, q=A, qs=512, k=A, v=A, slot=16384, slots=4, sl=A, lens=A, batch=2, most=128, out=A, os_=512):
    return _lib()[1].lfm_attention_decode(sh or _shape(), q, qs, k, v, slot, slots, sl, lens, batch, most, 0, 0, None,
                                          out, os_, None)


def shared(sh=None, pk=A, pv=A, pctx=64, prefix=64, q=A, k=A, lens=A, batch=2, most=128, work=A, nbytes=1 << 40):
    return _lib()[1].lfm_attention_shared(sh or _shape(), q, 512, pk, pv, pctx, prefix, k, A, 16384, 4, A, lens, batch,
                                          most, A, 512, work, nbytes, None)


S = 1 << 30


def evict(sh=None, src=(S, 2 * S, 3 * S, 4 * S), dst=(5 * S, 6 * S, 7 * S, 8 * S), slot=16384, slots=4, sl=9 * S,
          lens=10 * S, out=11 * S, batch=2, most=128, budget=16, first=2, last=2):
    return _lib()[1].lfm_cache_evict(sh or _shape(), *src, *dst, slot, slots, sl, lens, out, batch, most, budget, first,
                                     last, None)


@pytest.mark.parametrize("kw", BAD_SHAPES)
@pytest.mark.parametrize("call", [window, weights, decode, shared])
def test_bad_shapes(call, kw):
    assert call(sh=_shape(**kw)) == 1
    assert "lfm_attention_" in _lib()[1].lfm_ops_error().decode()


@pytest.mark.parametrize("kw", BAD_SHAPES[:6])
def test_bad_shapes_of_an_eviction(kw):
    assert evict(sh=_shape(**kw)) == 1


@pytest.mark.parametrize("call,kw", [
    (window, dict(q=None)), (window, dict(q=A + 8)), (window, dict(qs=504)), (window, dict(qs=514)),
    (window, dict(k=None)), (window, dict(v=A + 2)), (window, dict(n=0)), (window, dict(start=125)),
    (window, dict(start=0xffffffff)), (window, dict(n=(1 << 20) + 1, sh="long")), (window, dict(out=None)),
    (window, dict(os_=500)), (window, dict(sh="bf16", qs=516)), (weights, dict(lse=None)), (weights, dict(acc=None)),
    (weights, dict(k=A + 4)), (weights, dict(n=129)),
    (decode, dict(lens=None)), (decode, dict(batch=0)), (decode, dict(batch=65536)), (decode, dict(slots=0)),
    (decode, dict(sl=None, batch=5)), (decode, dict(slot=16380)), (decode, dict(slot=16376)), (decode, dict(most=129)),
    (decode, dict(k=None)), (decode, dict(v=A + 1)), (decode, dict(out=A + 4)),
    (shared, dict(pk=None)), (shared, dict(pv=A + 8)), (shared, dict(prefix=65)), (shared, dict(pctx=(1 << 24) + 1)),
    (shared, dict(work=None)), (shared, dict(work=A + 4)), (shared, dict(nbytes=15)), (shared, dict(lens=None)),
    (evict, dict(src=(None, 2 * S, 3 * S, 4 * S))), (evict, dict(src=(S, 2 * S, None, 4 * S))),
    (evict, dict(dst=(5 * S, 6 * S, 7 * S, None))), (evict, dict(out=None)), (evict, dict(out=10 * S + 4)),
    (evict, dict(out=9 * S)), (evict, dict(budget=0)), (evict, dict(first=10, last=7)),
    (evict, dict(first=0xffffffff, last=0xffffffff)), (evict, dict(dst=(S, 6 * S, 7 * S, 8 * S))),
    (evict, dict(dst=(S + 64, 6 * S, 7 * S, 8 * S))), (evict, dict(dst=(5 * S, S, 7 * S, 8 * S))),
    (evict, dict(dst=(5 * S, 5 * S, 7 * S, 8 * S))), (evict, dict(dst=(S, 2 * S, 3 * S, 8 * S))),
    (evict, dict(dst=(5 * S, 6 * S, 3 * S, 8 * S))), (evict, dict(src=(S, S, 3 * S, 4 * S), dst=(S, S, 3 * S, 4 * S))),
    (evict, dict(most=200)), (evict, dict(batch=0)),
])
def test_refusals(call, kw):
    kw = dict(kw)
    if kw.get("sh") == "long":
        kw["sh"] = _shape(ctx=1 << 24)
    elif kw.get("sh") == "bf16":
        kw["sh"] = _shape(dtype=2)
    assert call(**kw) == 1
    assert len(_lib()[1].lfm_ops_error()) > 20


def test_status_and_workspace():
    _, lib = _lib()
    assert lib.lfm_attention_status(None, None) == 1
    assert lib.lfm_attention_shared_workspace(_shape(), 0, 64) == 0
    assert lib.lfm_attention_shared_workspace(_shape(heads=7), 4, 64) == 0
    assert lib.lfm_attention_shared_workspace(_shape(), 4, 64) > 0


def test_shape_layout_matches_c_and_rust(tmp_path):
    m, _ = _lib()
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = [f for f, _ in m.AttnShape._fields_]
    src = tmp_path / "shape.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "lfm_cuda.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu\\n", offsetof(lfm_attn_shape, {f}));\n' for f in names) +
        '  printf("%zu\\n", sizeof(lfm_attn_shape));\n  return 0;\n}\n')
    exe = tmp_path / "shape"
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [getattr(m.AttnShape, f).offset for f in names] + [ctypes.sizeof(m.AttnShape)]
    rs = open(os.path.join(PKG, "rust", "lfm2-cuda-sys", "src", "lib.rs")).read()
    body = re.search(r"pub struct lfm_attn_shape\s*\{(.*?)\}", rs, re.S).group(1)
    assert re.findall(r"pub (\w+):", body) == names
