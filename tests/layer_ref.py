"""64-bit restatement of the layer operators (numpy), for their tests: Philox
masks, activations and slopes, the forward pass and the gradients."""
import math

import numpy as np
from scipy.special import erfc, expit

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon et al., SC 2011) on arrays of uint64 holding 32-bit words."""
    low = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    c = [np.asarray(w, np.uint64) for w in counter]
    k = [int(w) for w in key]
    for _ in range(rounds):
        p0 = np.uint64(0xD2511F53) * c[0]
        p1 = np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k[0]), p1 & low,
             (p0 >> s32) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def keep_mask(m, n, p, seed, offset):
    blocks = (n + 7) // 8
    col, row = np.meshgrid(np.arange(blocks), np.arange(m))
    words = philox4x32((col, row, np.full_like(col, offset & 0xFFFFFFFF),
                        np.full_like(col, offset >> 32)), (seed & 0xFFFFFFFF, seed >> 32))
    r16 = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=2)
    return r16.reshape(m, blocks * 8)[:, :n] >= threshold(p)


def drop(v, spec):
    """D(v); spec = (p, seed, offset) or None."""
    if spec is None or threshold(spec[0]) == 0:
        return v
    t = threshold(spec[0])
    if t == 65536:
        return np.zeros_like(v)
    with np.errstate(invalid="ignore"):
        return np.where(keep_mask(*v.shape, *spec), v * (65536.0 / (65536 - t)), 0.0)


def act(z, name):
    if name == "relu":
        return np.where(z > 0, z, 0.0)
    if name == "gelu":
        return z * 0.5 * erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z * expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * expit(z)
    return z


def slope(z, name):
    if name == "relu":
        return np.where(z > 0, 1.0, 0.0)
    if name == "gelu":
        return 0.5 * erfc(-z / math.sqrt(2)) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        g = expit(c * (z + 0.044715 * z ** 3))
        return g + z * g * (1 - g) * c * (1 + 3 * 0.044715 * z ** 2)
    if name == "silu":
        g = expit(z)
        return g + z * g * (1 - g)
    return np.ones_like(z)


def linear(x, w, bias, act_name, spec, residual):
    z = x @ w.T
    if bias is not None:
        z = z + bias
    out = drop(act(z, act_name), spec)
    return (out if residual is None else residual + out), z


def linear_grad(dy, x, w, pre, act_name, spec):
    dz = drop(dy, spec)
    if act_name != "none":
        dz = dz * slope(pre, act_name)
    return dz @ w, dz.T @ x, dz.sum(0), dz
