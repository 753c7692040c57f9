"""Plain forms of the operators on rows of logits, in numpy, and the error
bounds of their 32-bit kernels.

Inputs are numpy arrays of the values that the kernels see (bf16 inputs
already rounded), and the temperature is the fp32 number that the C entry
points take.  ``rules`` is the definition in 32-bit steps, each rounded by
itself, so a kernel's result is equal to it bit for bit; everything else is in
64 bits.  Bounds count roundings: U = 2^-24 is half a step of fp32 relative to
the value.
"""

import numpy as np

U = 2.0 ** -24
INF = np.inf


def allowed_bits(words, classes):
    """[n, ceil(classes / 32)] int32 words -> [n, classes] booleans."""
    w = words.astype(np.int64) & 0xFFFFFFFF
    return ((w[:, :, None] >> np.arange(32)) & 1).reshape(w.shape[0], -1)[:, :classes].astype(bool)


def table_rows(index, n, rows):
    if index is None:
        return np.zeros(rows, np.int64) if n == 1 else np.arange(rows)
    i = np.asarray(index, np.int64)
    return np.where((i >= 0) & (i < n), i, -1)


def counts(history, offsets, rows, classes):
    n = np.zeros((rows, classes), np.int64)
    for r in range(rows):
        lo = min(max(int(offsets[r]), 0), len(history))
        hi = min(max(int(offsets[r + 1]), lo), len(history))
        h = history[lo:hi]
        h = h[(h >= 0) & (h < classes)]
        np.add.at(n[r], h, 1)
    return n


def rules(x, bias=None, row_bias=None, masks=None, row_mask=None, history=None, history_offsets=None,
          repetition=None, frequency=None, presence=None, dtype=np.float32):
    """The rules in steps of ``dtype``: float32 is what the kernels compute."""
    with np.errstate(all="ignore"):
        y = x.astype(dtype)
        rows, classes = y.shape
        if history is not None:
            n = counts(history, history_offsets, rows, classes)
            one = np.ones(rows, dtype)
            r = (one if repetition is None else repetition.astype(dtype))[:, None]
            f = (0 * one if frequency is None else frequency.astype(dtype))[:, None]
            p = (0 * one if presence is None else presence.astype(dtype))[:, None]
            z = np.where(y > 0, y / r, y * r) - (f * n.astype(dtype) + p)
            y = np.where(n > 0, z, y)
        if bias is not None:
            t = table_rows(row_bias, bias.shape[0], rows)
            y = np.where((t >= 0)[:, None], y + bias[t].astype(dtype), y)
        if masks is not None:
            t = table_rows(row_mask, masks.shape[0], rows)
            y = np.where((t >= 0)[:, None] & ~allowed_bits(masks, classes)[t], dtype(-INF), y)
        return y


def sort_keys(x, last_ties=False):
    """Order of the classes of each row, best first: NaN, then values down, equal
    values by class."""
    v = np.where(np.isnan(x), INF, x)
    c = np.arange(x.shape[1])
    out = np.empty(x.shape, np.int64)
    for r in range(x.shape[0]):
        out[r] = np.lexsort((-c if last_ties else c, -v[r], ~np.isnan(x[r])))
    return out


def lse(x, axis=-1):
    with np.errstate(all="ignore"):
        m = np.max(x, axis=axis, keepdims=True) if x.shape[axis] else np.full(x.shape[:-1] + (1,), -INF)
        low = np.where(np.isfinite(m), m, 0.0)
        return np.log(np.sum(np.exp(x - low), axis=axis)) + np.squeeze(low, axis)


def sum_error(x, tau):
    """Relative error of a kernel's sum of exp((x - max) / tau) over the last
    axis (terms in fp32, -inf ones absent): a term's argument has one rounding
    of the difference, one of the scale 1 / tau and one of the product, the
    hardware exponential is within a step (2 U), and a thread's partial sum of
    its elements rounds at each addition; partial sums join in 64 bits.  Threads
    hold whole packs of up to eight elements and one of the row's last: 256 of
    them or more, 64 in rows of up to 2048 classes, of which at most 64 are
    entries that the sum leaves out."""
    with np.errstate(all="ignore"):
        d = (np.max(x, axis=-1, keepdims=True) - x) / tau
        e = np.where(np.isfinite(d), np.exp(-np.where(np.isfinite(d), d, 0)), 0.0)
        d = np.where(np.isfinite(d), d, 0.0)
        own = np.sum(e * (3 * d + 4), -1) / np.maximum(np.sum(e, -1), 1e-300)
        classes = x.shape[-1] + 64
        threads = 64 if x.shape[-1] <= 2048 else 256
        return (own + 8 * -(-classes // (8 * threads)) + 1) * U


def top(x, k, tau, last_ties=False):
    """values, indices, rest of rows after the rules (float32), rest in 64 bits."""
    tau = float(np.float32(tau))
    rows, classes = x.shape
    order = sort_keys(x, last_ties)
    values = np.full((rows, k), -INF, np.float32)
    indices = np.full((rows, k), -1, np.int32)
    n = min(k, classes)
    values[:, :n] = np.take_along_axis(x, order[:, :n], 1)
    indices[:, :n] = np.where(values[:, :n] == -INF, -1, order[:, :n])
    others = np.take_along_axis(x, order[:, n:], 1).astype(np.float64)
    rest = lse(others / tau) if n < classes else np.full(rows, -INF)
    error = (sum_error(others, tau) if n < classes else np.zeros(rows)) + 2 * U * np.abs(np.where(np.isfinite(rest), rest, 0))
    return values, indices, rest, error


def teacher_entries(values, indices, classes):
    """Which entries count: a class of the row's, not -inf, the first of its class."""
    ok = (indices >= 0) & (indices < classes) & ~(values == -INF)
    for r in range(indices.shape[0]):
        seen = set()
        for j in range(indices.shape[1]):
            if ok[r, j] and indices[r, j] in seen:
                ok[r, j] = False
            elif ok[r, j]:
                seen.add(int(indices[r, j]))
    return ok


def distill(x, values, indices, rest, tau, grad_loss=None):
    """Loss, state and gradient in 64 bits, and their error bounds."""
    tau = float(np.float32(tau))
    rows, classes = x.shape
    x = x.astype(np.float64)
    ok = teacher_entries(values, indices, classes)
    loss, grad = np.zeros(rows), np.zeros((rows, classes))
    state = np.zeros((rows, 4))
    loss_err, grad_err, state_err = np.zeros(rows), np.zeros((rows, classes)), np.zeros((rows, 4))
    g = np.ones(rows) if grad_loss is None else grad_loss.astype(np.float64)
    with np.errstate(all="ignore"):
        for r in range(rows):
            if not ok[r].any():
                continue
            at = indices[r][ok[r]].astype(np.int64)
            t = np.append(values[r][ok[r]].astype(np.float64) / tau, -INF if rest is None else np.float64(rest[r]))
            logq = t - lse(t)
            q = np.exp(logq)
            entry = np.zeros(classes, bool)
            entry[at] = True
            others = x[r][~entry]
            m = x[r].max()
            mr = others.max() if len(others) else -INF
            low = mr if np.isfinite(mr) or np.isnan(mr) else 0.0
            zr = np.sum(np.exp((others - low) / tau)) if mr != -INF else 0.0
            er = sum_error(others[None], tau)[0] if mr != -INF else 0.0
            z = np.sum(np.exp((x[r] - (m if m != -INF else 0.0)) / tau)) if m != -INF else 0.0
            state[r] = m, z, mr, zr
            state_err[r] = 0, (er + 4 * U) * z, 0, (er + U) * zr
            if m == -INF:
                loss[r] = INF
                continue
            # Relative to the maximum: next to the lowest value a log would vanish.
            logz = np.log(z)
            logp = np.append((x[r][at] - m) / tau, np.log(zr) + (low - m) / tau if zr > 0 else -INF) - logz
            loss[r] = tau * tau * np.sum(np.where(q > 0, q * (logq - logp), 0.0))
            # The rest's sum enters each log p through the whole, and the rest's once more.
            loss_err[r] = tau * tau * 2 * er + 2 * U * abs(loss[r]) + 1e-12
            p = np.exp((x[r] - m) / tau - logz)
            # The rest's shares of itself: far below the entries they still add up to one.
            own = np.where(entry | (x[r] == -INF), 0.0, np.exp((x[r] - low) / tau) / zr if zr > 0 else 0.0)
            grad[r] = np.where(entry, 0.0, p - q[-1] * own)
            grad[r][at] = p[at] - q[:-1]
            grad[r] *= tau * g[r]
            # The exponential's argument and itself, the sums, a division and the scale.
            d = np.where(p > 0, np.abs(x[r] - m) / tau, 0.0)
            d0 = np.where(own > 0, np.abs(x[r] - low) / tau, 0.0)
            q_of = np.zeros(classes)
            q_of[at] = q[:-1]
            grad_err[r] = tau * abs(g[r]) * (p * ((3 * d + 8) * U + er) + q[-1] * own * ((3 * d0 + 8) * U + er) + 4 * U * q_of)
            grad_err[r] += 4 * U * np.abs(grad[r])
            grad_err[r] += tau * abs(g[r]) * 1e-37  # exponentials below the normal range may flush
    return loss, state, grad, loss_err, state_err, grad_err
