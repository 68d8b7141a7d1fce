"""How far a session-cache attention output may be from the 64-bit value in
norm, beside the elementwise worst cases of cache_attn_ref, and an emulation of
the kernels' number formats that shows what the limits catch."""

import math

import numpy as np

LOG2E = math.log2(math.e)
SHIFT = {"f32": 15.0, "f16": 15.0, "bf16": 0.0}


def plain32(q, k, v, scale):
    """softmax(scale q k^T) v for one row in numpy's fp32."""
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    s = (k @ q) * np.float32(scale)
    e = np.exp(s - s.max())
    return ((e @ v) / e.sum(dtype=np.float32)).astype(np.float64)


def fp16_floor(w, v, top):
    """What fp16's smallest step leaves of one row's output, in norm: a weight of 2^top times its share w of the
    largest is off by half a step of 2^-24 at most, whatever its size, and the errors of n keys add up as the norm of
    their value rows."""
    return 2.0 ** (-25 - top) * w.max() * float(np.linalg.norm(v[w > 0]))


def score_cut(d, s):
    """What the tensor core's sums cost a row's scores s (nats): each of the d / 16 products of 16 is added to a partial
    sum that is cut off, not rounded, to 24 bits, which loses less than 2^-23 of it. For the key that matters, the
    largest score, the partial sums grow to that score, and an error of its score is one of every other weight."""
    return d / 16 * 2.0 ** -23 * float(np.abs(s).max())


def limit(kind, plain_error, floor=0.0):
    """Relative error in norm that a call's rows may have, given that of the plain fp32 form on the same inputs.

    fp32 queries: every rounding of the kernels is at most four of fp32's (pairs carry 22 bits instead of 24, the
    exponential 2^-22 instead of 2^-24, tensor-core sums lose up to a whole step instead of half of one), so four
    times the plain form's error; beside it the distance from the shifted reference, up to 2^4 in log2 units with half
    a step of 2^-20 of its own, and the sums of a tile, cut off up to eight times at half a step of 2^-23 on average:
    2^-21 + 2^-21. 16 bits: the weight's and the output's half steps (2^-11, 2^-8 at most, each). `floor` is fp16_floor's share of the output's
    norm and score_cut's largest."""
    own = {"f32": 2.0 ** -20, "f16": 2 * 2.0 ** -11, "bf16": 2 * 2.0 ** -8}[kind]
    return 4 * plain_error + own + floor


def norm_error(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


def _halves(x, keep_low):
    hi = x.astype(np.float16).astype(np.float64)
    return hi + (x - hi).astype(np.float16).astype(np.float64) if keep_low else hi


def emulate_f32(q, k, v, scale, q_low=True, p_low=True, shift=SHIFT["f32"], to_size=True):
    """One row of fp32 queries as the kernels' number formats have it (sums in 64 bits): q, brought to size by a power
    of two (or only times the scores' scale), and the weights as fp16 pairs, of which a half can be left out, the weights relative to the maximum less
    `shift`."""
    by = 2.0 ** (13 - math.floor(math.log2(np.abs(q).max()))) if to_size else scale * LOG2E
    s = ((k @ _halves(q * by, q_low)).astype(np.float32) * np.float32(scale * LOG2E / by)).astype(np.float32)
    m = np.float32(s.max() - np.float32(shift))
    p = np.exp2((s - m).astype(np.float64)).astype(np.float32).astype(np.float64)
    return _halves(p, p_low) @ v / p.sum()


def dominated(rng, kind, heads, kv, n, d, nats, at):
    """Queries [heads][d], keys and values [kv][n][d] (64-bit values that the types hold): key `at` of each KV head is
    `nats` above every other key for all of its queries, and its value row is 0, so the output is what the other
    weights make of the other rows. Values are large enough that fp16 outputs are not subnormal."""
    qt, ct = {"f32": (np.float32, np.float16), "f16": (np.float16, np.float16)}.get(kind, (None, None))

    def to(x, t):
        if t is not None:
            return x.astype(t).astype(np.float64)
        import torch
        return torch.from_numpy(x).to(torch.bfloat16).double().numpy()

    q = np.repeat(to(rng.normal(0, 1, (kv, d)), qt), heads // kv, 0)
    k, v = to(rng.normal(0, 1, (kv, n, d)), ct), to(rng.normal(0, 32, (kv, n, d)), ct)
    for h in range(kv):
        x = q[h * (heads // kv)]
        want = (k[h] @ x * d ** -0.5).max() + nats
        k[h, at] = to(x * (want * math.sqrt(d) / (x @ x)), ct)
        v[h, at] = 0
    return q, k, v
