"""Plain 64-bit forms of the decoding operators, and the errors their float32
kernels may make."""

from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # half a step of float32, relative


def visible(rows, cols, length, window, sinks):
    """(rows, cols) bool: the keys that each query of a sequence of that length sees."""
    p = length - rows + np.arange(rows)[:, None]
    j = np.arange(cols)[None]
    seen = j <= p
    if window is not None:
        seen &= (j > p - window) | (j < sinks)
    return seen


def attention(q, k, v, lengths, window, sinks, scale):
    """Of (batch, heads, rows, features) float32 arrays, in 64 bits; and the bound
    of a float32 kernel's error, for each output row."""
    batch, heads, rows, features = q.shape
    share = heads // k.shape[1]
    out = np.zeros(q.shape)
    bound = np.zeros((batch, heads, rows, 1))
    for b in range(batch):
        seen = visible(rows, k.shape[2], int(lengths[b]), window, sinks)
        n = seen.sum(-1)
        for h in range(heads):
            qq, kk, vv = q[b, h].astype(float), k[b, h // share].astype(float), v[b, h // share].astype(float)
            for i in range(rows):
                if not n[i]:
                    continue
                ks, vs = kk[seen[i]], vv[seen[i]]
                s = ks @ qq[i] * scale
                w = np.exp(s - s.max())
                out[b, h, i] = w @ vs / w.sum()
                # A score is a sum of `features` products, each of factors held to 2^-22
                # or better (16 EPS) and added in some order (features EPS), times a
                # rounded scale. An error d of the scores moves every weight by at most a
                # factor exp(d), both in the sum and in the weights. Sixteen lanes or
                # more share the keys, so a chain of sums is at most n / 16 + 16 long;
                # exp2 is good to 2 EPS, the rescalings and the quotient to a few more.
                d = abs(scale) * (np.abs(ks) @ np.abs(qq[i])).max() * (features + 24) * EPS
                bound[b, h, i] = (2 * d + (2 * (n[i] / 16 + 16) + 32) * EPS) * np.abs(vs).max()
    return out, bound


def bfloat_down(x):
    """float32 towards -inf to bfloat16, as float32."""
    bits = x.view(np.uint32).astype(np.int64)
    cut = bits // 65536 * 65536
    return np.where((cut != bits) & (x < 0), cut + 65536, cut).astype(np.uint32).view(np.float32)


def bfloat_up(x):
    return -bfloat_down(-x) + np.float32(0)


def cache_rows(x):
    """Rows of a 4-bit cache (int32) of float32 (..., features), group by group
    from the format's description."""
    features = x.shape[-1]
    groups = features // 32
    code = np.zeros((*x.shape[:-1], features // 2), np.uint8)
    words = np.zeros((*x.shape[:-1], groups), np.uint32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = x[..., 32 * g:32 * g + 32]
            low = bfloat_down(part.min(-1) + np.float32(0))
            step = bfloat_up((part.max(-1) - low) * np.float32(1 / 15))
            lost = ~np.isfinite(part).all(-1) | ~np.isfinite(low) | ~np.isfinite(step)
            q = np.rint((part - low[..., None]) / step[..., None])
            q = np.where((step[..., None] > 0) & ~lost[..., None], np.clip(q, 0, 15), 0).astype(np.uint8)
            word = (low.view(np.uint32) & np.uint32(0xffff0000)) | (step.view(np.uint32) >> np.uint32(16))
            words[..., g] = np.where(lost, np.uint32(0x7fc07fc0), word)
            for n in range(16):
                code[..., n * groups + g] = q[..., n] | (q[..., n + 16] << 4)
    return np.concatenate([code.view(np.int32), words.view(np.int32)], -1)


def cache_values(rows, features):
    """What cache rows stand for, in 64 bits."""
    groups = features // 32
    code = rows[..., :features // 8].copy().view(np.uint8)
    words = rows[..., features // 8:].copy().view(np.uint32)
    out = np.zeros((*rows.shape[:-1], features))
    for g in range(groups):
        low = (words[..., g] & np.uint32(0xffff0000)).view(np.float32).astype(float)
        step = (words[..., g] << np.uint32(16)).view(np.float32).astype(float)
        for n in range(16):
            byte = code[..., n * groups + g]
            out[..., 32 * g + n] = low + step * (byte & 15)
            out[..., 32 * g + 16 + n] = low + step * (byte >> 4)
    return out


def beam_candidates(logits, scores, finished=None, eos=None):
    """(batch, beams, vocabulary) scores of all candidates, in 64 bits."""
    x = logits.astype(float)
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        total = np.exp(x - np.where(np.isfinite(top), top, 0)).sum(-1, keepdims=True)
        out = x - (np.where(np.isfinite(top), top, 0) + np.log(np.where(np.isneginf(top), 1, total)))
    out = out + scores.astype(float)[..., None]
    if finished is not None:
        end = np.full(x.shape, -np.inf)
        end[..., eos] = scores
        out = np.where(finished[..., None], end, out)
    return out


def beam_best(logits, scores, count, finished=None, eos=None):
    x = beam_candidates(logits, scores, finished, eos)
    batch, _, vocabulary = x.shape
    flat = x.reshape(batch, -1)
    order = np.argsort(-flat, -1, kind="stable")[:, :count]
    return (np.take_along_axis(flat, order, -1), (order // vocabulary).astype(np.int32),
            (order % vocabulary).astype(np.int32))
