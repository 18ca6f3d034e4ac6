"""Distillation from a teacher's top tokens stated in binary64 numpy, one row at a time: the
definition the device results are held to (see rsc_distill in the C header)."""

import numpy as np


def inverse(temperature: float) -> np.float32:
    return np.float32(1.0) / np.float32(temperature)


def row(x, ids, y, temperature=1.0, tail=False):
    """(loss, d loss / d x, p * mass + r * tail, t) of one row, the last two as vectors over the
    vocabulary: the magnitudes that the gradient is a difference of. x binary32, ids and y the
    row's entries."""
    s = inverse(temperature)
    with np.errstate(over="ignore", invalid="ignore"):
        v = (x.astype(np.float32) * s).astype(np.float64)
    here = (ids >= 0) & (ids < len(x)) & (y != -np.inf)
    ids, y = ids[here].astype(np.int64), y[here].astype(np.float64)
    zero = np.zeros(len(x))
    if len(ids) == 0:
        return 0.0, zero, zero, zero
    with np.errstate(all="ignore"):
        m = v.max()
        e = np.exp(v - m)
        total = e.sum()
        if not total > 0:
            total = np.nan
        p = e / total
        logp = v - m - np.log(total)
        if tail:
            logt = y
            t = np.exp(y)
            r, mass = max(0.0, 1.0 - t.sum()), max(1.0, t.sum())
        else:
            top = y.max()
            t = np.exp(y - top)
            logt = y - top - np.log(t.sum())
            t = t / t.sum()
            r, mass = 0.0, 1.0
        loss = np.where(t == 0, 0.0, t * (logt - logp[ids])).sum()
        # The unlisted tokens by themselves, against their own maximum: their share of the row may
        # be far below what binary64 holds.
        listed = np.zeros(len(x), bool)
        listed[ids] = True
        rest = np.zeros(len(x))
        if r > 0:
            log_rest = -np.inf  # against m: as such it would swallow the sums' logs where m is large
            if (~listed).any() and v[~listed].max() != -np.inf:
                mr = v[~listed].max()
                er = np.exp(v[~listed] - mr)
                rest[~listed] = er / er.sum()
                log_rest = (mr - m) + np.log(er.sum())
            loss = loss + r * (np.log(r) - log_rest + np.log(total))
        dense = np.zeros(len(x))
        np.add.at(dense, ids, t)
        grad = p * mass - r * rest - dense
    return float(loss), float(s) * grad, p * mass + r * rest, dense


def batch(x, ids, y, n, temperature=1.0, tail=False):
    """Rows of arrays: losses, gradients, magnitudes, teacher probabilities."""
    cap = ids.shape[1]
    out = [row(x[i], ids[i, :min(cap, n[i] if n is not None else cap)],
               y[i, :min(cap, n[i] if n is not None else cap)], temperature, tail)
           for i in range(len(x))]
    return [np.array([o[k] for o in out]) for k in range(4)]
