"""Plain restatements in 64 bits of the feed-forward half of a layer (numpy, CPU): residual and norm with codes, routing, experts."""
import numpy as np


def add_norm(x, residual, weight, eps, offset):
    """(h in x's type, v = h (offset + w), 1 / rms), rows of x."""
    h = x if residual is None else (x.astype(np.float64) + residual.astype(np.float64)).astype(x.dtype)
    h64 = h.astype(np.float64)
    v = h64 * (offset + weight.astype(np.float64)) if weight is not None else h64
    return h, v, 1 / np.sqrt((h64 * h64).mean(-1, keepdims=True) + eps)


def codes(v, rstd, symmetric):
    """(codes, scale, zero point) of v rstd."""
    if symmetric:
        top = np.abs(v).max(-1, keepdims=True)
        span, low, most, shift = top, np.zeros_like(top), 127.0, 0
    else:
        low = v.min(-1, keepdims=True)
        span, most, shift = v.max(-1, keepdims=True) - low, 255.0, 128
    q = np.floor((v - low) * most / np.where(span > 0, span, 1.0) + 0.5)
    q = np.where(span > 0, q - shift, 0.0)
    return q.astype(np.int8), span / most * rstd, (low + span * (128 / 255.0)) * rstd if not symmetric else np.zeros_like(low)


def route(logits, bias, top_k, sigmoid, groups, top_groups, group_best, renormalise, factor):
    """(ids, weights): of equal values the larger logit first, then the lower number."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max)) + 0.0
    n, e = x.shape
    ids, weights = np.full((n, top_k), -1, np.int32), np.zeros((n, top_k))
    for t in range(n):
        row = x[t]
        there = row > -np.inf
        if not there.any():
            continue
        with np.errstate(over="ignore", under="ignore"):
            score = 1 / (1 + np.exp(-row)) if sigmoid else np.exp(row - row.max())
        if not sigmoid:
            score = score / score.sum()
        value = np.where(there, score + (0 if bias is None else bias.astype(np.float64)), -np.inf)
        value = np.where(np.isnan(value), -np.inf, value)
        if groups > top_groups:
            per = value.reshape(groups, -1)
            best = np.sort(per, 1)[:, ::-1][:, :group_best].sum(1)
            keep = np.argsort(-best, kind="stable")[:top_groups]
            out = np.ones(groups, bool)
            out[keep] = False
            value = np.where(np.repeat(out, e // groups), -np.inf, value)
        order = np.lexsort((np.arange(e), -row, -value))[:top_k]
        order = order[value[order] > -np.inf]
        ids[t, :len(order)] = order
        w = score[order]
        if renormalise:
            logit = row[order]
            small = np.exp(logit - logit.max())  # what does not vanish, for scores that all do
            w = w / w.sum() if w.sum() > 1e-280 else small / small.sum()
        weights[t, :len(order)] = factor * w
    return ids, weights


def gated(gate, up, gelu):
    with np.errstate(over="ignore"):
        if gelu:
            return 0.5 * gate * (1 + np.tanh(np.sqrt(2 / np.pi) * (gate + 0.044715 * gate ** 3))) * up
        return gate / (1 + np.exp(-gate)) * up


def experts(x, ids, weights, first, second, residual, gelu):
    """first [E][2 f][d] (gate, up alternating), second [E][d][f] dequantised.  (out, (carried, before)): what relative errors act on,
    of the gated values and behind them, and of the weights and sums ahead of the gate (there the worst case, every error one way)."""
    x = x.astype(np.float64)
    out = np.zeros_like(x) if residual is None else residual.astype(np.float64)
    carried, before = np.abs(out), np.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = ids[t, j]
            if not 0 <= e < first.shape[0]:
                continue
            w, gu = abs(float(weights[t, j])), first[e] @ x[t]
            h = gated(gu[0::2], gu[1::2], gelu)
            out[t] += float(weights[t, j]) * (second[e] @ h)
            carried[t] += w * (np.abs(second[e]) @ np.abs(h))
            # neither gate is steeper than 1.13
            reach = np.abs(first[e]) @ np.abs(x[t])
            reach = reach[0::2] * (1.13 * np.abs(gu[1::2])) + reach[1::2] * np.abs(gated(gu[0::2], 1.0, gelu))
            before[t] += w * (np.abs(second[e]) @ reach)
    return out, (carried, before)


def experts_bound(want, size, many):
    """fp16 roundings (2^-11 of the value): of the gated product and of the result; with many rows also of every weight, and of each
    expert's output.  32-bit sums, exp and divisions are 2^-17 of what they act on at most (512 roundings of partial sums, halved).
    Below 2^-14 fp16 is spaced 2^-24."""
    carried, before = size
    half, sums = 2.0 ** -11, 2.0 ** -17
    return half * np.abs(want) + carried * ((3.1 if many else 1.1) * half + sums) + before * ((1.1 * half if many else 0.0) + sums) + 2.0 ** -16


def pack(codes_, bits):
    """Codes [outputs][inputs] in blocks of 4 inputs x 4 outputs, q + 8 / q + 128."""
    o, i = codes_.shape
    b = codes_.reshape(o // 4, 4, i // 4, 4).transpose(2, 0, 3, 1).reshape(-1).astype(np.int64)
    if bits == 8:
        return (b + 128).astype(np.uint8)
    return ((b[0::2] + 8) | (b[1::2] + 8) << 4).astype(np.uint8)


def matrix(rng, o, i, bits, block):
    """(packed, scales [groups][o] fp16, dequantised [o][i] in 64 bits)."""
    q = np.clip(np.rint(rng.standard_normal((o, i)) * (2.6 if bits == 4 else 40)), -8 if bits == 4 else -128, 7 if bits == 4 else 127)
    groups = i // block if block else 1
    scales = (np.exp(0.3 * rng.standard_normal((groups, o))) / ((2.6 if bits == 4 else 40) * np.sqrt(i))).astype(np.float16)
    w = q * np.repeat(scales.astype(np.float64), i // groups, 0).T
    return pack(q, bits), scales, w
