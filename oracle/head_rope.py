"""The norm of each query / key head with the position rotation, and the rotation by positions of
several axes, in 64 bits on the host. Rows are [T, H, D]; the first R = cos.shape[1] dims are rotated."""

import numpy as np


def axis_of(sections, interleaved=False):
    """The axis of each frequency: block after block, or the axes in turn while they have some left."""
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections)
    left, out = list(sections), []
    while sum(left):
        for a in range(len(sections)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return np.asarray(out)


def axes_cos_sin(positions, inv_freq, sections, interleaved=False):
    """cos, sin [T, R] of positions [axes, T] and inv_freq [R / 2]."""
    ang = np.asarray(positions, dtype=np.float64)[axis_of(sections, interleaved)].T * inv_freq.astype(np.float64)
    ang = np.concatenate([ang, ang], 1)
    return np.cos(ang), np.sin(ang)


def _partner(x, R):
    """(x[j + R/2], x[j - R/2]) swapped halves of the rotated dims, the rest 0."""
    out = np.zeros_like(x)
    out[..., :R // 2], out[..., R // 2:R] = x[..., R // 2:R], x[..., :R // 2]
    return out


def _full(cos, sin, D):
    """cos, sin [T, 1, D]: 1 and 0 behind R."""
    T, R = cos.shape
    c, s = np.ones((T, 1, D)), np.zeros((T, 1, D))
    c[:, 0, :R], s[:, 0, :R] = cos, sin
    return c, s


def forward(x, w, eps, cos, sin):
    """(rotated [T, H, D], magnitude of the terms) of x [T, H, D]; w None: no norm."""
    D, R = x.shape[-1], cos.shape[1]
    c, s = _full(np.asarray(cos, np.float64), np.asarray(sin, np.float64), D)
    y = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    sign = np.where(np.arange(D) < R // 2, -1.0, 1.0)
    z = _partner(y, R)
    return y * c + sign * z * s, np.abs(y) * np.abs(c) + np.abs(z) * np.abs(s)


def backward(g, x, w, eps, cos, sin):
    """(dx, magnitude, dw or None, its magnitude) from the gradient g [T, H, D] and the input x."""
    D, R = g.shape[-1], cos.shape[1]
    c, s = _full(np.asarray(cos, np.float64), np.asarray(sin, np.float64), D)
    sign = np.where(np.arange(D) < R // 2, 1.0, -1.0)
    z = g * c + sign * _partner(g * s, R)
    m = np.abs(g * c) + np.abs(_partner(g * s, R))
    if w is None:
        return z, m, None, None
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dw, mdw = (z * x * r).sum((0, 1)), (m * np.abs(x * r)).sum((0, 1))
    z, m = z * w, m * np.abs(w)
    return (r * (z - x * r * r * (z * x).mean(-1, keepdims=True)),
            r * (m + np.abs(x) * r * r * (m * np.abs(x)).mean(-1, keepdims=True)), dw, mdw)
