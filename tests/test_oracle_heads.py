"""The float64 statements of oracle/heads.py against library routines and differences (CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import heads as oh


def _rng(seed):
    return np.random.default_rng(seed)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotation_is_a_rotation(layout):
    """Products of two rotated heads depend on the distance of their positions only; norms of pairs stay."""
    r = _rng(1)
    freq = 10000.0 ** (-np.arange(8) / 8)
    x, y = r.normal(size=(2, 1, 1, 1, 20))
    at = lambda t, p: oh.rotate(t, np.array([p]), freq, 1.0, layout)
    d1 = (at(x, 7) * at(y, 3)).sum()
    d2 = (at(x, 1007) * at(y, 1003)).sum()
    assert abs(d1 - d2) < 1e-9
    a, b = oh.pair_columns(16, layout)
    z = at(x, 5)
    np.testing.assert_allclose(z[..., a] ** 2 + z[..., b] ** 2, x[..., a] ** 2 + x[..., b] ** 2, rtol=1e-12)
    np.testing.assert_array_equal(z[..., 16:], x[..., 16:])
    quarter = oh.rotate(np.eye(16)[None, :, None, :], np.ones(16), np.full(8, np.pi / 2), 1.0, layout)
    np.testing.assert_allclose(quarter[0, a, 0, b], 1.0, atol=1e-15)       # the first axis turns onto the second


def test_norm_against_torch_and_differences():
    r = _rng(2)
    x, w, g = r.normal(size=(2, 3, 2, 10)), r.normal(size=10), r.normal(size=(2, 3, 2, 10))
    freq, pos = r.uniform(0.1, 1, 4), np.arange(3)
    ref = torch.nn.functional.rms_norm(torch.tensor(x), (10,), torch.tensor(w), 1e-6).numpy()
    np.testing.assert_allclose(oh.norm_rotate(x, w, pos, None), ref, rtol=1e-10)
    f = lambda x, w: (g * oh.norm_rotate(x, w, pos, freq, 1.3, "interleaved", 1e-3)).sum()
    dx, dw = oh.norm_rotate_grads(x, w, g, pos, freq, 1.3, "interleaved", 1e-3)
    ux, uw, h = r.normal(size=x.shape), r.normal(size=10), 1e-6
    np.testing.assert_allclose((f(x + h * ux, w) - f(x - h * ux, w)) / (2 * h), (dx * ux).sum(), rtol=1e-7)
    np.testing.assert_allclose((f(x, w + h * uw) - f(x, w - h * uw)) / (2 * h), (dw * uw).sum(), rtol=1e-7)


def test_cross_attention_against_torch():
    r = _rng(3)
    q, k, v = r.normal(size=(2, 5, 4, 6)), r.normal(size=(2, 7, 2, 6)), r.normal(size=(2, 7, 2, 6))
    live = r.random((2, 7)) < 0.7
    live[:, 0] = True
    out, lse = oh.cross_attention(q, k, v, live, 0.3)
    tq, tk, tv = (torch.tensor(t).permute(0, 2, 1, 3) for t in (q, np.repeat(k, 2, 2), np.repeat(v, 2, 2)))
    ref = torch.nn.functional.scaled_dot_product_attention(tq, tk, tv, torch.tensor(live)[:, None, None], scale=0.3)
    np.testing.assert_allclose(out, ref.permute(0, 2, 1, 3).numpy(), rtol=1e-10, atol=1e-12)
    s = (tq @ tk.transpose(-1, -2) * 0.3).masked_fill(~torch.tensor(live)[:, None, None], -np.inf)
    np.testing.assert_allclose(lse, torch.logsumexp(s, -1).numpy(), rtol=1e-12)


def test_cross_attention_gradients_against_differences_and_dead_keys():
    r = _rng(4)
    q, k, v = r.normal(size=(2, 3, 4, 5)), r.normal(size=(2, 6, 2, 5)), r.normal(size=(2, 6, 2, 5))
    g = r.normal(size=q.shape)
    live = np.array([[1, 1, 0, 1, 0, 1], [0] * 6], bool)
    grads = oh.cross_attention_grads(q, k, v, live, g)
    f = lambda q, k, v: (g * oh.cross_attention(q, k, v, live)[0]).sum()
    h = 1e-6
    for i, t in enumerate((q, k, v)):
        u = r.normal(size=t.shape)
        args = [[q, k, v], [q, k, v]]
        args[0][i], args[1][i] = t + h * u, t - h * u
        np.testing.assert_allclose((f(*args[0]) - f(*args[1])) / (2 * h), (grads[i] * u).sum(), rtol=1e-6)
    out, lse = oh.cross_attention(q, k, v, live)
    assert not out[1].any() and np.isneginf(lse[1]).all()
    assert not any(t[1].any() for t in grads)
    assert not grads[1][0, ~live[0]].any() and not grads[2][0, ~live[0]].any()
    k2, v2 = k.copy(), v.copy()
    k2[~live], v2[~live] = np.nan, np.inf
    np.testing.assert_array_equal(oh.cross_attention(q, k2, v2, live)[0], out)
