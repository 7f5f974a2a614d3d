"""Oracle: root-mean-square norm behind a residual's addition, in float64.  TEST INFRASTRUCTURE ONLY.

The stream h is given: the sum x + r, rounded to the stream's type as the program that adds first has it.
"""

from __future__ import annotations

import numpy as np


def rms_norm(h, w=None, eps=1e-6):
    h = np.asarray(h, np.float64)
    return h / np.sqrt(np.mean(h * h, -1, keepdims=True) + eps) * (1.0 if w is None else np.asarray(w, np.float64))


def rms_norm_grads(h, gy, gh=None, w=None, eps=1e-6):
    """(dh, dw) of sum(gy y) + sum(gh h)."""
    h, gy = np.asarray(h, np.float64), np.asarray(gy, np.float64)
    i = 1.0 / np.sqrt(np.mean(h * h, -1, keepdims=True) + eps)
    n, gn = h * i, gy * (1.0 if w is None else np.asarray(w, np.float64))
    dh = i * (gn - n * np.mean(gn * n, -1, keepdims=True)) + (0.0 if gh is None else np.asarray(gh, np.float64))
    return dh, (gy * n).reshape(-1, h.shape[-1]).sum(0)


def scales(y, group=0):
    """A scale for each group of columns (0: the row): max(max |y|, 2^-100) / 448."""
    y = np.asarray(y, np.float64)
    y = y.reshape(*y.shape[:-1], -1, group or y.shape[-1])
    return np.maximum(np.abs(y).max(-1), 2.0 ** -100) / 448.0
