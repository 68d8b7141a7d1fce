"""Attention over session caches, measured operator by operator.

Five operators of the library that serve sessions whose caches outgrow or
share their context, each with a plain torch form beside the library's call:

  window   lfm_attention_window    prompt attention, sliding window + sink positions, row statistics
  decode   lfm_attention_decode    one token of each session, window + sinks, optional accumulated weights
  shared   lfm_attention_shared    one token of each session over one shared prefix + each session's own cache
  weights  lfm_attention_weights   a prompt's attention weight summed per cache position
  evict    lfm_cache_evict         keep sinks, recent and heaviest positions of a cache, in order

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run`
makes one pass, in plain torch (`own` false) or through the library.

Types: "f32" is fp32 queries and outputs over fp16 caches (the engine's own
layout), "f16" and "bf16" have queries, outputs and caches in that type.
Caches are [slot][kv head][position][head_dim].
"""

import ctypes
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"f32": (torch.float32, torch.float16, 0), "f16": (torch.float16, torch.float16, 1),
          "bf16": (torch.bfloat16, torch.bfloat16, 2)}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The last 64-token chunk of a 4096-position session streamed through the
        # engine's chunked prompt path, with a window: the latency of a short call.
        dict(name="window_chunk", op="window", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=4096, start=4032,
             n=64, window=1024, sinks=4, pad=512),
        # The engine's long prompt (3840 tokens, q inside fused q|k rows), windowed.
        dict(name="window_prompt", op="window", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=4096, start=0,
             n=3840, window=1024, sinks=4, pad=512),
        # A long document in 16-bit types with wide heads and a window that no tile divides.
        dict(name="window_long", op="window", type="bf16", heads=32, kv_heads=8, head_dim=128, ctx=8200, start=0,
             n=8192, window=1500, sinks=5, pad=0),
        # One session's decode step at the engine's benchmark depth, weights accumulated: latency.
        dict(name="decode_one", op="decode", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=4096, batch=1,
             slots=1, min_len=577, max_len=577, window=0, sinks=0, acc=True, pad=512),
        # 64 sessions decoded together, as lfm_batch_decode does, each seeing its window and sinks.
        dict(name="decode_window", op="decode", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=4096, batch=64,
             slots=64, min_len=129, max_len=4096, window=1024, sinks=4, acc=False, pad=512),
        # Long ragged sessions in fp16, six query heads to a KV head, weights accumulated for eviction.
        dict(name="decode_long", op="decode", type="f16", heads=48, kv_heads=8, head_dim=128, ctx=32768, batch=24,
             slots=26, min_len=1000, max_len=32768, window=0, sinks=0, acc=True, pad=0),
        # A few sessions behind one system prompt.
        dict(name="shared_few", op="shared", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=1024, batch=4,
             slots=4, prefix=1000, min_len=0, max_len=129, pad=512),
        # Many short answers over one long document, eight query heads to a KV head.
        dict(name="shared_many", op="shared", type="bf16", heads=32, kv_heads=4, head_dim=128, ctx=512, batch=256,
             slots=256, prefix=16384, min_len=1, max_len=512, pad=0),
        # The last 32 queries of a 3840-token prompt choose what the cache keeps.
        dict(name="weights_tail", op="weights", type="f32", heads=32, kv_heads=8, head_dim=64, ctx=4096, start=3808,
             n=32, window=0, sinks=0, pad=512),
        # Every query of a long prompt counts.
        dict(name="weights_prompt", op="weights", type="bf16", heads=32, kv_heads=8, head_dim=128, ctx=8192, start=0,
             n=8191, window=0, sinks=0, pad=0),
        # One full session cut to a quarter.
        dict(name="evict_one", op="evict", type="f32", kv_heads=8, head_dim=64, ctx=4096, batch=1, slots=1,
             min_len=4096, max_len=4096, budget=1024, keep_first=4, keep_last=256),
        # 48 long ragged sessions cut to a common budget, an odd one.
        dict(name="evict_many", op="evict", type="bf16", kv_heads=8, head_dim=128, ctx=8192, batch=48, slots=50,
             min_len=1500, max_len=8192, budget=2045, keep_first=4, keep_last=301),
    ]


def draw(rng):
    def spread(lo, hi):  # over the logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5))))

    kind = rng.choice(["f32", "f16", "bf16"])
    heads, kv = rng.choice([(32, 8), (8, 8), (24, 8), (20, 4), (48, 8), (28, 4), (32, 4), (6, 1), (16, 8)])
    d = rng.choice([64, 128])
    op = rng.choice(["window", "decode", "shared", "weights", "evict"])
    c = dict(op=op, type=kind, heads=heads, kv_heads=kv, head_dim=d)
    if op in ("window", "weights"):
        n = spread(1, 8000)
        start = rng.choice([0, spread(1, 8000)])
        while heads * n * (start + n) > 8 * 4000 * 8000:  # below the largest listed case
            n, start = (n + 1) // 2, start // 2
        c.update(start=start, n=n, ctx=start + n + rng.choice([0, spread(1, 300)]), pad=rng.choice([0, kv * d]),
                 window=rng.choice([0, spread(1, 4000), spread(64, 2000)]), sinks=rng.choice([0, 1, 4, spread(1, 200)]))
    elif op == "decode":
        batch = spread(1, 96)
        hi = min(spread(1, 30000), max(1, 24 * 30000 * 8 * 128 // (batch * kv * d)))
        c.update(batch=batch, slots=batch + rng.choice([0, 3]), ctx=hi + rng.choice([0, 7, 100]),
                 min_len=rng.choice([0, 1, hi]), max_len=hi, window=rng.choice([0, spread(1, hi)]),
                 sinks=rng.choice([0, 4, spread(1, 100)]), acc=rng.choice([True, False]), pad=rng.choice([0, kv * d]))
    elif op == "shared":
        batch, prefix = spread(1, 250), spread(1, 16000)
        while batch * heads * prefix * d > 256 * 32 * 16000 * 128:
            prefix = (prefix + 1) // 2
        hi = spread(1, 700)
        c.update(batch=batch, slots=batch + rng.choice([0, 2]), prefix=prefix, ctx=hi + rng.choice([0, 5, 64]),
                 min_len=rng.choice([0, 1, hi]), max_len=hi, pad=rng.choice([0, kv * d]))
    else:
        del c["heads"]
        batch = spread(1, 64)
        hi = min(spread(2, 16000), 48 * 8000 * 8 * 128 // (batch * kv * d))
        budget = rng.randint(1, hi)
        first = min(rng.choice([0, 1, 4, 33]), budget)
        c.update(batch=batch, slots=batch + rng.choice([0, 1]), ctx=hi + rng.choice([0, 9]), min_len=rng.choice([0, 1, hi]),
                 max_len=hi, budget=budget, keep_first=first, keep_last=rng.randint(0, budget - first))
    return c


def _lens(c):
    """The sessions' lengths: the first at the longest, the others spread over the case's range."""
    r = random.Random(c["batch"] * 1000003 + c["max_len"])
    return [c["max_len"]] + [r.randint(c["min_len"], c["max_len"]) for _ in range(c["batch"] - 1)]


def _seen(p, window, sinks):
    """How many positions a query at position p sees."""
    if not window or window > p:
        return p + 1
    return window + min(sinks, p + 1 - window)


def _is_seen(p, j, window, sinks):
    """Whether a query at position p sees position j (tensors that broadcast)."""
    see = j <= p
    if window:
        see = see & ((p - j < window) | (j < sinks))
    return see


# ------------------------------------------------------------------ inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qt, ct, _ = _TYPES[c["type"]]
    kv, d = c["kv_heads"], c["head_dim"]

    def normal(*shape, dtype=ct):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    st = {"case": c}
    if c["op"] in ("window", "weights"):
        n, heads = c["n"], c["heads"]
        st["q"] = 1.5 * normal(n, heads * d + c["pad"], dtype=qt)
        st["k"], st["v"] = normal(1, kv, c["ctx"], d), normal(1, kv, c["ctx"], d)
        st["out"] = torch.empty(n, heads * d, device="cuda", dtype=qt)
        st["lse"] = torch.empty(n, heads, device="cuda")
        st["acc"] = torch.zeros(1, kv, c["ctx"], device="cuda")
        if c["op"] == "weights":  # the prompt's attention has left its row statistics
            st["lse"].copy_(_window_plain(st)[1])
        return st
    batch, slots = c["batch"], c["slots"]
    order = torch.randperm(slots, generator=g, device="cuda")[:batch]
    st["slots"] = order.to(torch.int32)
    st["lens"] = torch.tensor(_lens(c), device="cuda", dtype=torch.int32)
    st["k"], st["v"] = normal(slots, kv, c["ctx"], d), normal(slots, kv, c["ctx"], d)
    if c["op"] == "evict":
        # few positions carry most of the weight; some were never looked at
        w = torch.exp(2.5 * normal(slots, kv, c["ctx"], dtype=torch.float32)) * 1e-2
        st["acc"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.05, torch.zeros_like(w), w)
        st["pos"] = torch.arange(c["ctx"], device="cuda", dtype=torch.int32).expand(slots, kv, c["ctx"]).contiguous()
        for k in ("k", "v", "acc", "pos"):
            st[k + "_out"] = torch.zeros_like(st[k])
        st["lens_out"] = torch.zeros_like(st["lens"])
        return st
    st["q"] = 1.5 * normal(batch, c["heads"] * d + c["pad"], dtype=qt)
    st["out"] = torch.empty(batch, c["heads"] * d, device="cuda", dtype=qt)
    if c["op"] == "decode":
        earlier = torch.rand(slots, kv, c["ctx"], generator=g, device="cuda") * (c["heads"] / kv / c["max_len"])
        st["acc"] = earlier if c["acc"] else None  # of about one step before this one
    else:
        st["pk"], st["pv"] = normal(kv, c["prefix"], d), normal(kv, c["prefix"], d)
        most = (c["prefix"] + 127) // 128
        st["work"] = torch.empty(4 * batch * c["heads"] * (d + 2) * min(most, 64), device="cuda", dtype=torch.uint8)
    return st


# ------------------------------------------------------------- plain forms
def _softmax_parts(s, see):
    """exp(s - max) over the seen positions, their sum and the maximum; a row that sees none has sum 0."""
    s = s.masked_fill_(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    e = s.sub_(m).exp_()
    return e, e.sum(-1, keepdim=True), m


def _window_scores(st):
    c = st["case"]
    n, heads, kv, d = c["n"], c["heads"], c["kv_heads"], c["head_dim"]
    end = c["start"] + n
    q = st["q"][:, :heads * d].float().view(n, kv, heads // kv, d).permute(1, 0, 2, 3).reshape(kv, -1, d)
    s = (q * d ** -0.5) @ st["k"][0, :, :end].float().transpose(1, 2)
    p = torch.arange(c["start"], end, device="cuda").view(n, 1, 1)
    see = _is_seen(p, torch.arange(end, device="cuda"), c["window"], c["sinks"])
    return s.view(kv, n, heads // kv, end), see


def _window_plain(st):
    c = st["case"]
    n, heads, kv, d = c["n"], c["heads"], c["kv_heads"], c["head_dim"]
    s, see = _window_scores(st)
    e, l, m = _softmax_parts(s, see)
    o = e.view(kv, -1, e.shape[-1]) @ st["v"][0, :, :c["start"] + n].float()
    o = o.view(kv, n, heads // kv, d) / l
    lse = (m + l.log()).squeeze(-1)
    return o.permute(1, 0, 2, 3).reshape(n, heads * d).to(st["out"].dtype), lse.permute(1, 0, 2).reshape(n, heads)


def _weights_plain(st):
    c = st["case"]
    n, heads, kv = c["n"], c["heads"], c["kv_heads"]
    s, see = _window_scores(st)
    lse = st["lse"].view(n, kv, heads // kv).permute(1, 0, 2).unsqueeze(-1)
    w = s.sub_(lse).exp_().masked_fill_(~see, 0.0)
    st["acc"][0, :, :c["start"] + n] += w.sum((1, 2))
    return st["acc"]


def _own_scores(st):
    """Scores of each session's one query over its own cache [batch][kv][g][position], and which it sees."""
    c = st["case"]
    heads, kv, d, most = c["heads"], c["kv_heads"], c["head_dim"], c["max_len"]
    q = st["q"][:, :heads * d].float().view(-1, kv, heads // kv, d) * d ** -0.5
    k = st["k"][st["slots"].long(), :, :most].float()
    j, end = torch.arange(most, device="cuda"), st["lens"].view(-1, 1, 1, 1)
    return q, q @ k.transpose(2, 3), _is_seen(end - 1, j, c.get("window", 0), c.get("sinks", 0))


def _decode_plain(st):
    c = st["case"]
    at = st["slots"].long()
    _, s, see = _own_scores(st)
    e, l, _ = _softmax_parts(s, see)
    w = e / torch.where(l > 0, l, torch.ones_like(l))
    o = w @ st["v"][at, :, :c["max_len"]].float()
    if st["acc"] is None:
        return o.reshape(o.shape[0], -1).to(st["out"].dtype), None
    st["acc"][at, :, :c["max_len"]] += w.sum(2)
    return o.reshape(o.shape[0], -1).to(st["out"].dtype), st["acc"]


def _shared_plain(st):
    c = st["case"]
    kv, d, g = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    q, s, see = _own_scores(st)
    batch = q.shape[0]
    rows = q.permute(1, 0, 2, 3).reshape(kv, batch * g, d)
    sp = (rows @ st["pk"].float().transpose(1, 2)).view(kv, batch, g, -1).permute(1, 0, 2, 3)
    every = torch.ones(1, dtype=torch.bool, device="cuda").expand(batch, 1, 1, c["prefix"])
    e, l, _ = _softmax_parts(torch.cat((sp, s), -1), torch.cat((every, see), -1))
    ep = e[..., :c["prefix"]].permute(1, 0, 2, 3).reshape(kv, batch * g, -1)
    o = (ep @ st["pv"].float()).view(kv, batch, g, d).permute(1, 0, 2, 3)
    o = o + e[..., c["prefix"]:] @ st["v"][st["slots"].long(), :, :c["max_len"]].float()
    return (o / l).reshape(batch, -1).to(st["out"].dtype)


def _evict_plain(st):
    c = st["case"]
    at, most, budget = st["slots"].long(), c["max_len"], c["budget"]
    lens = st["lens"].view(-1, 1, 1)
    j = torch.arange(most, device="cuda")
    w = st["acc"][at, :, :most].clone()
    always = (j < c["keep_first"]) | (j >= lens - c["keep_last"]) | (lens <= budget)
    w = torch.where(always, torch.full_like(w, math.inf), w)
    w = torch.where(j >= lens, torch.full_like(w, -math.inf), w)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]  # equal weights: the earlier position
    kept = torch.sort(torch.where(first < lens, first, most), -1).values
    real = kept < most
    kept = torch.where(real, kept, 0)
    for k in ("acc", "pos", "k", "v"):
        src = st[k][at, :, :most]
        i, ok = (kept, real) if src.dim() == 3 else (kept.unsqueeze(-1).expand(*kept.shape, src.shape[-1]), real.unsqueeze(-1))
        old = st[k + "_out"][at, :, :i.shape[2]]
        st[k + "_out"][at, :, :i.shape[2]] = torch.where(ok, src.gather(2, i), old)
    st["lens_out"].copy_(st["lens"].clamp(max=budget))
    return {k: st[k] for k in ("k_out", "v_out", "acc_out", "pos_out", "lens_out")}


# ------------------------------------------------------- the library's calls
_lib = None


def _library():
    global _lib
    if _lib is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm2-w9100-rust_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import lfm2_b200
        _lib = (lfm2_b200, lfm2_b200.lib())
    return _lib


def _at(t):
    return None if t is None else t.data_ptr()


def _own_run(st):
    m, lib = _library()
    c = st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    shape = st.get("shape")
    if shape is None:  # the caller's plan, made once per model
        shape = st["shape"] = ctypes.byref(m.AttnShape(_TYPES[c["type"]][2], c.get("heads", c["kv_heads"]), c["kv_heads"],
                                                       c["head_dim"], c["ctx"], 0.0))
    op = c["op"]
    if op == "window":
        q, out = st["q"], st["out"]
        m.ops_check(lib.lfm_attention_window(shape, q.data_ptr(), q.stride(0), _at(st["k"]), _at(st["v"]), c["start"],
                                             c["n"], c["window"], c["sinks"], out.data_ptr(), out.stride(0),
                                             _at(st["lse"]), stream), op)
        return out, st["lse"]
    if op == "weights":
        q = st["q"]
        m.ops_check(lib.lfm_attention_weights(shape, q.data_ptr(), q.stride(0), _at(st["k"]), c["start"], c["n"],
                                              c["window"], c["sinks"], _at(st["lse"]), _at(st["acc"]), stream), op)
        return st["acc"]
    slot = st["k"].stride(0)
    if op == "decode":
        q, out = st["q"], st["out"]
        m.ops_check(lib.lfm_attention_decode(shape, q.data_ptr(), q.stride(0), _at(st["k"]), _at(st["v"]), slot,
                                             c["slots"], _at(st["slots"]), _at(st["lens"]), c["batch"], c["max_len"],
                                             c["window"], c["sinks"], _at(st["acc"]), out.data_ptr(), out.stride(0),
                                             stream), op)
        return out, st["acc"]
    if op == "shared":
        q, out, work = st["q"], st["out"], st["work"]
        m.ops_check(lib.lfm_attention_shared(shape, q.data_ptr(), q.stride(0), _at(st["pk"]), _at(st["pv"]),
                                             c["prefix"], c["prefix"], _at(st["k"]), _at(st["v"]), slot, c["slots"],
                                             _at(st["slots"]), _at(st["lens"]), c["batch"], c["max_len"],
                                             out.data_ptr(), out.stride(0), work.data_ptr(), work.numel(), stream), op)
        return out
    m.ops_check(lib.lfm_cache_evict(shape, _at(st["k"]), _at(st["v"]), _at(st["acc"]), _at(st["pos"]), _at(st["k_out"]),
                                    _at(st["v_out"]), _at(st["acc_out"]), _at(st["pos_out"]), slot, c["slots"],
                                    _at(st["slots"]), _at(st["lens"]), _at(st["lens_out"]), c["batch"], c["max_len"],
                                    c["budget"], c["keep_first"], c["keep_last"], stream), op)
    return {k: st[k] for k in ("k_out", "v_out", "acc_out", "pos_out", "lens_out")}


_PLAIN = {"window": _window_plain, "weights": _weights_plain, "decode": _decode_plain, "shared": _shared_plain,
          "evict": _evict_plain}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["case"]["op"]](state)


# -------------------------------------------------------------- exact values
def _exact_rows(q, k, v, see):
    """softmax(q k^T / sqrt(d)) over the seen columns, in 64 bits: weights, output, log of the sum of exponentials."""
    x = torch.where(see, q @ k.mT / math.sqrt(q.shape[-1]), -math.inf)
    lse = torch.logsumexp(x, -1)
    w = torch.where(torch.isinf(lse).unsqueeze(-1), 0.0, torch.exp(x - lse.unsqueeze(-1)))
    return w, None if v is None else w @ v, lse


def exact(c, seed):
    st = prepare(c, seed)
    kv, d = c["kv_heads"], c["head_dim"]
    if c["op"] == "evict":
        outs = {k: torch.zeros_like(st[k]) for k in ("k_out", "v_out", "acc_out", "pos_out")}
        slots, lens = st["slots"].tolist(), st["lens"].tolist()
        for b, (slot, n) in enumerate(zip(slots, lens)):
            for h in range(kv):
                if n <= c["budget"]:
                    kept = torch.arange(n, device="cuda")
                else:
                    lo, hi = c["keep_first"], n - c["keep_last"]
                    key = st["acc"][slot, h, lo:hi].double()
                    middle = torch.argsort(-key, dim=0, stable=True)[:c["budget"] - lo - c["keep_last"]].sort().values + lo
                    kept = torch.cat((torch.arange(lo, device="cuda"), middle, torch.arange(hi, n, device="cuda")))
                for k in ("k", "v", "acc", "pos"):
                    outs[k + "_out"][slot, h, :len(kept)] = st[k][slot, h].index_select(0, kept)
        outs["lens_out"] = torch.tensor([min(n, c["budget"]) for n in lens], dtype=torch.int32, device="cuda")
        return {k: v.double() if v.is_floating_point() else v for k, v in outs.items()}
    heads = c["heads"]
    g = heads // kv
    q = st["q"][:, :heads * d].double().unflatten(1, (heads, d))
    if c["op"] in ("window", "weights"):
        n, end = c["n"], c["start"] + c["n"]
        see = _is_seen(torch.arange(c["start"], end, device="cuda")[:, None], torch.arange(end, device="cuda")[None],
                       c["window"], c["sinks"])
        out, lse = torch.zeros_like(q), torch.zeros(n, heads, dtype=torch.float64, device="cuda")
        acc = st["acc"].double()
        for h in range(heads):
            k, v = st["k"][0, h // g, :end].double(), st["v"][0, h // g, :end].double()
            if c["op"] == "weights":  # the given statistics, not fresh ones
                x = q[:, h] @ k.mT / math.sqrt(d) - st["lse"][:, h, None].double()
                acc[0, h // g, :end] += torch.where(see, torch.exp(x), 0.0).sum(0)
            else:
                _, out[:, h], lse[:, h] = _exact_rows(q[:, h], k, v, see)
        return acc if c["op"] == "weights" else (out.flatten(1), lse)
    out = torch.zeros_like(q)
    acc = st["acc"].double() if c["op"] == "decode" and c["acc"] else None
    for b, (slot, n) in enumerate(zip(st["slots"].tolist(), st["lens"].tolist())):
        k, v = st["k"][slot, :, :n].double(), st["v"][slot, :, :n].double()
        if c["op"] == "shared":
            k, v = torch.cat((st["pk"].double(), k), 1), torch.cat((st["pv"].double(), v), 1)
            see = torch.ones(k.shape[1], dtype=torch.bool, device="cuda")
        else:
            see = _is_seen(n - 1, torch.arange(n, device="cuda"), c["window"], c["sinks"])
        if k.shape[1] == 0:
            continue
        w, o, _ = _exact_rows(q[b].view(kv, g, d), k, v, see)
        out[b] = o.reshape(heads, d)
        if acc is not None:
            acc[slot, :, :n] += w.sum(1)
    return out.flatten(1) if c["op"] == "shared" else (out.flatten(1), acc)


# ---------------------------------------------------------------------- work
def work(c):
    qb = 4 if c["type"] == "f32" else 2
    kv, d, heads = c["kv_heads"], c["head_dim"], c.get("heads", 0)
    if c["op"] in ("window", "weights"):
        start, n, window, sinks = c["start"], c["n"], c["window"], c["sinks"]
        pairs = sum(_seen(p, window, sinks) for p in range(start, start + n))
        first = max(0, start - window + 1) if window else 0
        rows = start + n - first + min(sinks, first)  # cache positions that some query sees
        if c["op"] == "weights":
            return {"bytes": n * heads * (d * qb + 4) + rows * kv * (2 * d + 8), "flops": 2 * pairs * heads * d}
        return {"bytes": n * heads * (2 * d * qb + 4) + rows * kv * 4 * d, "flops": 4 * pairs * heads * d}
    lens = _lens(c)
    if c["op"] == "evict":
        kept = sum(min(n, c["budget"]) for n in lens)
        weighed = sum(n for n in lens if n > c["budget"])
        return {"bytes": kv * (weighed * 4 + kept * (2 * 2 * 2 * d + 8 + 8)), "flops": 0}
    io = c["batch"] * heads * d * 2 * qb
    if c["op"] == "decode":
        seen = sum(_seen(n - 1, c["window"], c["sinks"]) for n in lens if n)
        return {"bytes": io + seen * kv * (4 * d + (8 if c["acc"] else 0)), "flops": 4 * seen * heads * d}
    seen = sum(lens)
    return {"bytes": io + (c["prefix"] + seen) * kv * 4 * d, "flops": 4 * (c["prefix"] * c["batch"] + seen) * heads * d}
