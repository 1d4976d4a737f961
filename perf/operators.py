"""What is measured of the layer operators: a linear layer with bias,
activation, dropout and residual in one pass (``kernels.linear``), its
gradient (``kernels.linear_grad``) and dropout on its own
(``kernels.dropout``, ``kernels.dropout_grad``).

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits, rounded once at the end) or, where ``own`` is true, by the calls a
user makes.  ``exact`` is the same in 64 bits from the definitions.

Definitions, with rows m, outputs n, and ``drop`` = (p, seed, offset):

    z[m,n]    = sum_k x[m,k] w[n,k] + bias[n]
    out[m,n]  = residual[m,n] + D(act(z))[m,n]
    D(v)[m,n] = keep[m,n] ? v * 65536 / (65536 - t) : 0,  t = round(65536 p)
    keep[m,n] = r16[m,n] >= t
    r16[m,n]  = 16 bits number n % 8 (low half first) of the four words of
                Philox4x32-10 (Salmon et al., 2011) at the counter
                (n / 8, m, offset low, offset high), key (seed low, seed high)

    dz = D(dy) * act'(z);  dx = dz w;  dw = dz^T x;  db[n] = sum_m dz[m,n]
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, op, dtype, m, k, n, act="none", p=0.0, residual=False, bias=True, pre=False,
          pitched=False, w_t=False):
    """``pitched``: the activations are columns of a wider buffer; ``w_t``:
    the weight is kept as [k, n] and passed as its transpose."""
    c = {"op": op, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "p": p,
         "residual": residual, "bias": bias, "pre": pre, "pitched": pitched, "w_t": w_t}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # serving one sample through a 4096-wide layer: the weight is read once
        _case("linear_token_bf16", "linear", "bf16", 1, 4096, 4096, "gelu"),
        # serving a handful of rows that arrived together, block's second layer
        _case("linear_few_f16", "linear", "f16", 24, 8192, 2048, "none", residual=True),
        # the small MLP's hidden layer in training: 784 -> 128, batch 256
        _case("linear_small_f32", "linear", "f32", 256, 784, 128, "relu", p=0.1, pre=True),
        # a ragged last batch through layers of odd widths
        _case("linear_ragged_bf16", "linear", "bf16", 1531, 1019, 777, "gelu_tanh", p=0.2,
              residual=True, pre=True),
        # the wide MLP's layer: 4096 -> 4096, batch 8192
        _case("linear_wide_f32", "linear", "f32", 8192, 4096, 4096, "relu", p=0.1, pre=True),
        # a feed-forward block's first layer in training: four times as wide
        _case("linear_wide_bf16", "linear", "bf16", 16384, 4096, 16384, "gelu", p=0.1, pre=True),
        # the gradients of the layers above
        _case("grad_small_f32", "linear_grad", "f32", 256, 784, 128, "relu", p=0.1, pre=True),
        _case("grad_ragged_f16", "linear_grad", "f16", 2047, 1003, 1531, "silu", p=0.1, pre=True),
        _case("grad_wide_f32", "linear_grad", "f32", 8192, 4096, 4096, "relu", p=0.1, pre=True),
        _case("grad_wide_bf16", "linear_grad", "bf16", 16384, 4096, 16384, "gelu", p=0.1, pre=True),
        # dropout between layers: the small MLP's activations, and a block's
        # output added to its input
        _case("dropout_small_f32", "dropout_grad", "f32", 256, 1, 128, p=0.5),
        _case("dropout_wide_bf16", "dropout", "bf16", 16384, 1, 16384, p=0.1, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "linear_grad", "dropout", "dropout_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    p = rng.choice([0.0, 0.1, rng.uniform(0.01, 0.9)])
    if op in ("dropout", "dropout_grad"):
        p = p or 0.1
        m, n = _log(rng, 1, 16384), _log(rng, 16, 16384)
        return _case("", op, dtype, m, 1, n, p=p, residual=op == "dropout" and rng.random() < 0.5,
                     pitched=rng.random() < 0.25)
    k, n = _log(rng, 64, 8192), _log(rng, 64, 16384)
    if rng.random() < 0.5:  # half the layers have widths that are multiples of 64
        k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
    most = (16384 * 4096 * 16384 if dtype != "f32" else 8192 * 4096 * 4096) // (k * n)
    m = _log(rng, 1, max(1, min(16384, most)))
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op == "linear":
        return _case("", op, dtype, m, k, n, act, p, residual=rng.random() < 0.5,
                     bias=rng.random() < 0.75, pre=rng.random() < 0.5,
                     pitched=rng.random() < 0.25, w_t=rng.random() < 0.25)
    return _case("", op, dtype, m, k, n, act, p, pre=act != "none", pitched=rng.random() < 0.25,
                 w_t=rng.random() < 0.25)


def _normal(gen, rows, cols, dt, scale=1.0, pitched=False):
    wide = cols + 24 if pitched else cols
    t = torch.empty((rows, wide), dtype=dt, device="cuda").normal_(0.0, scale, generator=gen)
    return t[:, 8:8 + cols] if pitched else t


def prepare(case, seed):
    """Normal activations, Kaiming-normal weights, pre-activations of the size
    such a layer gives, gradients of a mean loss's size (times the scale a
    16-bit training loop applies)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    m, k, n = case["m"], case["k"], case["n"]
    # the dropout stream a training loop keeps: its seed, and a call counter
    s = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 64),
         "offset": seed % 1000 + (1 << 33)}
    if case["op"] in ("dropout", "dropout_grad"):
        s["x"] = _normal(gen, m, n, dt, 1.0, case["pitched"])
        s["residual"] = _normal(gen, m, n, dt) if case["residual"] else None
        return s
    s["x"] = _normal(gen, m, k, dt, 1.0, case["pitched"])
    scale = math.sqrt(2.0 / k)
    s["w"] = _normal(gen, k, n, dt, scale).t() if case["w_t"] else _normal(gen, n, k, dt, scale)
    if case["op"] == "linear":
        s["bias"] = _normal(gen, 1, n, dt, 0.1)[0] if case["bias"] else None
        s["residual"] = _normal(gen, m, n, dt) if case["residual"] else None
    else:
        s["pre"] = _normal(gen, m, n, dt, 1.4) if case["pre"] else None
        s["dy"] = _normal(gen, m, n, dt, 0.05, case["pitched"])
    return s


# ---- plain form -----------------------------------------------------------------


def _mulhilo(mult, a):
    """High and low 32 bits of mult * a, held in int64: a in 16-bit halves."""
    low = mult * (a & 0xFFFF)
    mid = mult * (a >> 16) + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox(c0, c1, c2, c3, k0, k1):
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c0)
        h1, l1 = _mulhilo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _drop(v, case, state):
    """D(v) for float32 v [m, n]."""
    t = _threshold(case["p"])
    if t == 0:
        return v
    if t == 65536:
        return torch.zeros_like(v)
    m, n = v.shape
    seed, off = state["seed"], state["offset"]
    col = torch.arange((n + 7) // 8, device=v.device, dtype=torch.int64).view(1, -1).expand(m, -1)
    row = torch.arange(m, device=v.device, dtype=torch.int64).view(-1, 1).expand(-1, (n + 7) // 8)
    c2 = torch.full_like(col, off & 0xFFFFFFFF)
    words = _philox(col, row, c2, off >> 32, seed & 0xFFFFFFFF, seed >> 32)
    r16 = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=2)
    keep = r16.reshape(m, -1)[:, :n] >= t
    return torch.where(keep, v * (65536.0 / (65536 - t)), torch.zeros_like(v))


_R2 = math.sqrt(0.5)
_RPI = math.sqrt(2.0 / math.pi)
_PHI = 1.0 / math.sqrt(2.0 * math.pi)


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * (0.5 * (1.0 + torch.erf(z * _R2)))
    if act == "gelu_tanh":
        return z * (0.5 * (1.0 + torch.tanh(_RPI * (z + 0.044715 * z * z * z))))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * _R2)) + z * (_PHI * torch.exp(-0.5 * z * z))
    if act == "gelu_tanh":
        t = torch.tanh(_RPI * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * (_RPI * (1.0 + 0.134145 * z * z))
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain(state):
    case = state["case"]
    dt = _TYPES[case["dtype"]]
    if case["op"] in ("dropout", "dropout_grad"):
        y = _drop(state["x"].float(), case, state)
        if state["residual"] is not None:
            y = state["residual"].float() + y
        return y.to(dt)
    if case["op"] == "linear":
        z = state["x"].float() @ state["w"].float().t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
        out = _drop(_act(z, case["act"]), case, state)
        if state["residual"] is not None:
            out = state["residual"].float() + out
        return [out.to(dt), z.to(dt)] if case["pre"] else [out.to(dt)]
    dz = _drop(state["dy"].float(), case, state)
    if case["act"] != "none":
        dz = dz * _act_slope(state["pre"].float(), case["act"])
    return [(dz @ state["w"].float()).to(dt), (dz.t() @ state["x"].float()).to(dt),
            dz.sum(0).to(dt)]


def run(state):
    if not own:
        return _plain(state)
    from ferrograd_b200 import kernels
    case = state["case"]
    drop = kernels.Dropout(case["p"], state["seed"], state["offset"]) if case["p"] > 0 else None
    if case["op"] == "dropout":
        return kernels.dropout(state["x"], drop, residual=state["residual"])
    if case["op"] == "dropout_grad":
        return kernels.dropout_grad(state["x"], drop)
    if case["op"] == "linear":
        got = kernels.linear(state["x"], state["w"], state["bias"], act=case["act"],
                             residual=state["residual"], drop=drop, save_pre=case["pre"])
        return list(got) if case["pre"] else [got]
    return list(kernels.linear_grad(state["dy"], state["x"], state["w"], pre=state["pre"],
                                    act=case["act"], drop=drop))


# ---- in 64 bits -----------------------------------------------------------------


def _exact_keep(rows, n, t, seed, off, device):
    """keep for the given rows, from Philox's definition with the multipliers
    in 16-bit halves (every partial product below 2^48)."""
    blocks = (n + 7) // 8
    x = [torch.arange(blocks, device=device).repeat(len(rows)),
         rows.repeat_interleave(blocks),
         torch.full((len(rows) * blocks,), off % 2**32, device=device),
         torch.full((len(rows) * blocks,), off // 2**32, device=device)]
    key = [seed % 2**32, seed // 2**32]

    def product(a, c):
        part = a * (c % 65536)
        rest = a * (c // 65536) + part // 65536
        return rest // 65536, (rest % 65536) * 65536 + part % 65536

    for _ in range(10):
        hi_a, lo_a = product(x[0], 3528531795)
        hi_b, lo_b = product(x[2], 3449720151)
        x = [hi_b.bitwise_xor(x[1]).bitwise_xor(key[0]), lo_b,
             hi_a.bitwise_xor(x[3]).bitwise_xor(key[1]), lo_a]
        key = [(key[0] + 2654435769) % 2**32, (key[1] + 3144134277) % 2**32]
    keep = torch.empty((len(rows) * blocks, 8), dtype=torch.bool, device=device)
    for i in range(8):
        keep[:, i] = (x[i // 2] // 65536 ** (i % 2)) % 65536 >= t
    return keep.view(len(rows), blocks * 8)[:, :n]


def _exact_drop(v, case, state):
    t = math.floor(case["p"] * 65536 + 0.5)
    if t == 0:
        return v
    out = torch.zeros_like(v)
    if t < 65536:
        step = max(1, (1 << 25) // v.shape[1])
        for a in range(0, v.shape[0], step):
            rows = torch.arange(a, min(a + step, v.shape[0]), device=v.device)
            keep = _exact_keep(rows, v.shape[1], t, state["seed"], state["offset"], v.device)
            part = v[a:a + step] / (1.0 - t / 65536)
            out[a:a + step][keep] = part[keep]
    return out


def _exact_cdf(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda name: s[name].double()  # noqa: E731
    act = case["act"]
    if case["op"] in ("dropout", "dropout_grad"):
        y = _exact_drop(d("x"), case, s)
        return y if s["residual"] is None else y + d("residual")
    if case["op"] == "linear":
        z = torch.mm(d("x"), d("w").t())
        if s["bias"] is not None:
            z += d("bias")
        if act == "relu":
            a = z.clamp(min=0.0)
        elif act == "gelu":
            a = z * _exact_cdf(z)
        elif act == "gelu_tanh":
            a = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
        elif act == "silu":
            a = z * torch.sigmoid(z)
        else:
            a = z
        out = _exact_drop(a, case, s)
        if s["residual"] is not None:
            out = out + d("residual")
        return [out, z] if case["pre"] else [out]
    dz = _exact_drop(d("dy"), case, s)
    if act != "none":
        z = d("pre")
        if act == "relu":
            dz = torch.where(z > 0, dz, 0.0)
        elif act == "gelu":
            dz = dz * (_exact_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        elif act == "gelu_tanh":
            c = 2.0 * math.sqrt(2.0 / math.pi)
            g = torch.sigmoid(c * (z + 0.044715 * z ** 3))
            dz = dz * (g + z * g * (1 - g) * c * (1 + 3 * 0.044715 * z ** 2))
        else:
            g = torch.sigmoid(z)
            dz = dz * (g + z * g * (1 - g))
    return [torch.mm(dz, d("w")), torch.mm(dz.t(), d("x")), dz.sum(0)]


def work(case):
    e, m, k, n = _SIZE[case["dtype"]], case["m"], case["k"], case["n"]
    if case["op"] in ("dropout", "dropout_grad"):
        return {"bytes": e * m * n * (3 if case["residual"] else 2), "flops": 2 * m * n}
    if case["op"] == "linear":
        moved = (m * k + n * k + n * case["bias"]
                 + m * n * (1 + case["residual"] + case["pre"]))
        return {"bytes": e * moved, "flops": 2 * m * n * k}
    moved = m * n * (1 + case["pre"]) + 2 * m * k + 2 * n * k + n
    return {"bytes": e * moved, "flops": 4 * m * n * k}
