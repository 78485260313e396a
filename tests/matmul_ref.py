"""The products with packed weights in 64 bits, and bounds on how far a sum held in 32 bits may be from them.

Weights are decoded by the CPU oracle (the bits that the decode kernels are held to).  A kernel may split a weight into a
code and an offset, w = a * q + w0 with w0 the value of code 0, and add both parts up apart.  The tests' x are drawn with
independent signs around zero, so a partial sum of such terms spreads like
    R[t][r] = sqrt(sum over c of ((|w - w0| + |w0|) * x)^2)
and six times that is never met.  Each rounding is off by at most half a unit (2^-24) of the partial sum it ends, and all
that lie on the longest way of a product into the result are added up as if they had one sign: the sum over a sub-block (at
most 64), the two steps of scale and offset, two for every 512 elements of the row, 16 that join lanes, waves and pieces of
x, and the two roundings of the decoded weight that a kernel may leave out.  Where x and y are both 16-bit floats a kernel may
round x to 2^-17 of the largest of 32 neighbours; such errors have independent signs, spread like 2^-17 / sqrt(3) times about
2.5 R, below 1.2e-5 R, four tenths of the bound of the shortest sum, and get no allowance of their own.
"""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}       # the smallest step
# byte ranges of a block that hold codes (everything else: scales, minima)
CODES = {2: (2, 18), 3: (4, 20), 6: (2, 22), 7: (4, 24), 8: (2, 34), 9: (4, 36), 10: (16, 80), 11: (0, 96), 12: (16, 144), 13: (16, 176),
         14: (0, 192), 15: (2, 258), 20: (2, 18), 23: (8, 136)}


def decode(oracle, ty, packed, rows, cols):
    """(W, W0): the decoded matrix and its value at code 0, both in 64 bits."""
    w = oracle.dequantize(ty, packed).reshape(rows, cols).astype(np.float64)
    if ty in (1, 30):
        return w, np.zeros_like(w)
    bb = oracle.block_bytes(ty)
    z = packed.reshape(-1, bb).copy()
    lo, hi = CODES[ty]
    z[:, lo:hi] = 0
    return w, oracle.dequantize(ty, z.reshape(-1)).reshape(rows, cols).astype(np.float64)


def product(w, w0, x):
    """(y, bound) for x[t, cols] in 64 bits."""
    y = x @ w.T
    spread = np.sqrt(x ** 2 @ ((np.abs(w - w0) + np.abs(w0)) ** 2).T)
    steps = 64 + 2 + 2 * (w.shape[1] // 512 + 1) + 16 + 2
    return y, 6 * steps * U * spread


def outside(got, want, bound, kind):
    """How many values of `got` are further from `want` than `bound` and one rounding to the type allow."""
    tol = bound + HALF_STEP[kind] * (np.abs(want) + bound) + TINY[kind]
    return int(np.sum(~(np.abs(got.astype(np.float64) - want) <= tol)))


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def act(g, kind):
    if kind == "silu":
        return g * sigmoid(g)
    return 0.5 * g * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (g + 0.044715 * g ** 3)))


def moe(router, gate, up, down, x, top_k, gating, normalize, scale, activation):
    """gate, up, down: lists of (W, W0) per expert.  Returns (y, bound, ids, weights).  The bound follows each 32-bit
    rounding to the end; both activations have a slope of at most 1.13, and the exponential, the division and the
    products of an activation together are given 16 half units (GELU's argument g + 0.044715 g^3 may turn the error of a
    few half units into as many times 2 |z| of them, which matters only where the result has already saturated)."""
    logits = (x @ router.T).astype(np.float32)
    t_n, hidden = x.shape
    y, bound = np.zeros((t_n, hidden)), np.zeros((t_n, hidden))
    ids, weights = np.zeros((t_n, top_k), dtype=np.int32), np.zeros((t_n, top_k))
    for t in range(t_n):
        order = sorted(range(len(gate)), key=lambda e: (-logits[t, e], e))[:top_k]
        l = logits[t].astype(np.float64)
        p = np.exp(l - l.max()) / np.exp(l - l.max()).sum() if gating == "softmax" else sigmoid(l)
        w = p[order]
        w = (w / w.sum() if normalize else w) * scale
        ids[t], weights[t] = order, w
        for j, e in enumerate(order):
            g, dg = product(*gate[e], x[t:t + 1])
            u, du = product(*up[e], x[t:t + 1])
            a = act(g, activation)
            h = a * u
            # GELU: z = g * (sqrt(2/pi) + ...), tanh's argument is off by some half units of z: slope at most 1 / cosh^2
            da = 1.13 * dg + 16 * U * (np.abs(a) + (np.abs(g) if activation == "gelu" else 0.0))
            dh = da * np.abs(u) + (np.abs(a) + da) * du + 2 * U * np.abs(h)
            d, dd = product(*down[e], h)
            dd = dd + 6 * np.sqrt(dh ** 2 @ (down[e][0] ** 2).T)       # errors of independent sign
            # weight: exp of a difference of logits (each off by half a unit), a sum, two divisions, a product
            dw = (24 + len(gate)) * U * max(1.0, np.abs(l).max()) * abs(w[j])
            y[t] += w[j] * d[0]
            bound[t] += abs(w[j]) * dd[0] + dw * np.abs(d[0]) + (top_k + 16) * U * np.abs(w[j] * d[0])
    return y, bound, ids, weights
