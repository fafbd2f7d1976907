"""Norms of heads and rotary positions in 64 bits, element by element, for the tests of wd_kv_append_rope."""
import numpy as np


def frequencies(rotary, theta):
    return np.array([theta ** (-2.0 * p / rotary) for p in range(rotary // 2)])


def rotated(x, positions, freq, sections=(), neighbours=False, norm=None, eps=1e-6, factor=1.0):
    """x [rows][heads][dim]; positions [rows] or [rows][axes]; returns the same shape, and the size of what each element is made of."""
    x = np.array(x, np.float64)
    positions = np.asarray(positions, np.float64).reshape(x.shape[0], -1)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps) * np.asarray(norm, np.float64)
    y, size = x.copy(), np.abs(x)
    axis = [a for a, n in enumerate(sections) for _ in range(n)] or [0] * len(freq)
    for p, f in enumerate(freq):
        a, b = (2 * p, 2 * p + 1) if neighbours else (p, p + len(freq))
        angle = positions[:, axis[p]] * f
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y[:, :, a] = factor * (x[:, :, a] * c - x[:, :, b] * s)
        y[:, :, b] = factor * (x[:, :, b] * c + x[:, :, a] * s)
        size[:, :, a] = size[:, :, b] = abs(factor) * (np.abs(x[:, :, a]) + np.abs(x[:, :, b]))
    return y, size
