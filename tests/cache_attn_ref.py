"""64-bit plain forms of the session-cache attention operators, and the error
that each kernel may have on given inputs, for the tests."""

import ctypes
import math

import numpy as np

TYPES = {"f32": 0, "f16": 1, "bf16": 2}


def torch_types(kind):
    import torch
    return {"f32": (torch.float32, torch.float16), "f16": (torch.float16, torch.float16),
            "bf16": (torch.bfloat16, torch.bfloat16)}[kind]


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def seen(p, j, window, sinks):
    return (j <= p) & ((window == 0) | (p - j < window) | (j < sinks))


def attend(q, k, v, see, scale):
    """One query row q [d] over k, v [n][d] where `see`: output, log sum of exponentials, weights [n]."""
    w = np.zeros(k.shape[0])
    at = np.flatnonzero(see)
    if at.size == 0:
        return np.zeros(v.shape[1]), -math.inf, w
    s = k[at] @ q * scale
    m = s.max()
    e = np.exp(s - m)
    w[at] = e / e.sum()
    return w[at] @ v[at], m + math.log(e.sum()), w


def score_error(kind, q, k, scale):
    """Bound of a score's error: fp32 queries enter as an fp16 pair (hi off by 2^-11, the rest by 2^-11 of
    that, or by fp16's smallest step 2^-25), the cache as it is; d products are added in fp32, where an
    addition may be off by a step of 2^-23 of the largest partial sum (tensor cores cut off, they do not
    round); the scale and the change to powers of two are three more fp32 roundings."""
    qa, ka = np.abs(q).max(0) if q.ndim > 1 else np.abs(q), np.abs(k).max(0) if k.ndim > 1 else np.abs(k)
    size = float(np.sum(qa * ka)) * scale
    split = (2.0 ** -22 * size + 2.0 ** -25 * float(np.sum(ka))) if kind == "f32" else 0.0
    return split + (len(qa) * 2.0 ** -23 + 4 * 2.0 ** -24) * size


def out_error(kind, ds, n, vmax, out):
    """Bound of an output's error, given the bound ds of its scores: each weight is off by a factor of
    e^(2 ds) at most (its own score's and the sum's), the exponential by 2^-21, the weight as a tensor operand by half a
    step of its type (fp32: the pair's 2^-22 or 2^-25; 16 bits: eps / 2, and 2^-25 absolute in fp16), the n-term
    sums by n 2^-23 each, and the output is rounded to its type."""
    operand = {"f32": 2.0 ** -22 + n * 2.0 ** -25, "f16": 2.0 ** -11 + n * 2.0 ** -25, "bf16": 2.0 ** -8}[kind]
    out_step = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    rel = 2 * ds * (1 + ds) + 2.0 ** -20 + 2 * operand + 2 * (n + 8) * 2.0 ** -23
    return rel * vmax + out_step * np.abs(out) + (2.0 ** -25 if kind == "f16" else 0.0)
