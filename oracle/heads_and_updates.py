"""64-bit forms of two operators that the reference has no op for: heads normalised and rotated, and the orthogonal factor of a
matrix with the step along it (the formulas of include/autograd_b200.h, written plainly)."""
import numpy as np

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def rotate(x, c, s):
    """x (..., heads, D); c, s (..., rot / 2) of its tokens: columns i and i + rot / 2 turn by the angle of i."""
    h = c.shape[-1]
    y = np.array(x, np.float64)
    c, s = np.asarray(c, np.float64)[..., None, :], np.asarray(s, np.float64)[..., None, :]
    lo, hi = np.array(y[..., :h]), np.array(y[..., h:2 * h])
    y[..., :h] = lo * c - hi * s
    y[..., h:2 * h] = lo * s + hi * c
    return y


def _inv(x, eps):
    return 1.0 / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)


def heads(x, gamma, c, s, eps):
    """y = rotate(gamma * x / rms(x))"""
    x = np.asarray(x, np.float64)
    y = x * _inv(x, eps)
    return rotate(y if gamma is None else y * np.asarray(gamma, np.float64), c, s)


def heads_backward(dy, x, gamma, c, s, eps):
    """(dx, dgamma)"""
    x = np.asarray(x, np.float64)
    inv = _inv(x, eps)
    w = rotate(dy, c, -np.asarray(s))
    v = w if gamma is None else w * np.asarray(gamma, np.float64)
    dx = inv * (v - x * inv ** 2 * np.mean(v * x, -1, keepdims=True))
    return dx, (w * x * inv).reshape(-1, x.shape[-1]).sum(0)


def triples(coefficients, steps):
    return [tuple(coefficients)] * steps if np.ndim(coefficients) == 1 else [tuple(c) for c in coefficients]


def factor(u, coefficients=NEWTON_SCHULZ, steps=5, eps=1e-7):
    """X <- (a I + b X X^T + c (X X^T)^2) X from X = u / max(|u|, eps)."""
    x = np.asarray(u, np.float64)
    x = x / max(np.sqrt(np.sum(x * x)), eps)
    if x.shape[0] > x.shape[1]:
        return factor_steps(x.T, coefficients, steps).T
    return factor_steps(x, coefficients, steps)


def factor_steps(x, coefficients, steps):
    for a, b, c in triples(coefficients, steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def muon(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=1.0, grad_scale=1.0, steps=5,
         coefficients=NEWTON_SCHULZ, eps=1e-7):
    """(p, m, what the factor is taken of) after a step on one matrix"""
    p, g, m = (np.asarray(t, np.float64) for t in (p, g, m))
    g = g * grad_scale
    m = m + (1.0 - momentum) * (g - m)
    u = g + momentum * (m - g) if nesterov else m
    return p * (1.0 - lr * weight_decay) - lr * scale * factor(u, coefficients, steps, eps), m, u


def kept(x, bits):
    """x as the kernels keep it between products: 16-bit floats of x * 2^12 (11 significant bits, at least 2^-36 apart), or the sum
    of two of them (22 bits)."""
    y = (x * 4096.0).astype(np.float32)
    hi = y.astype(np.float16)
    if bits == 11:
        return hi.astype(np.float64) / 4096.0
    return (hi.astype(np.float64) + (y - hi.astype(np.float32)).astype(np.float16).astype(np.float64)) / 4096.0


def truncated(x):
    """x with 23 significant bits, cut off: what a sum in a tensor core keeps (the number with which 512 additions of one sign lose
    3e-5 of their sum, as they do)."""
    m, e = np.frexp(x)
    return np.ldexp(np.trunc(m * 2.0 ** 23), e - 23)


def product(x, y, bits):
    """x @ y of operands as they are kept: sums of 16 products are exact and truncated as they are added up, 128 elements at a time with
    22 bits, the products with a low part first; 32-bit sums of those."""
    high = [kept(v, 11) for v in (x, y)]
    low = [kept(v, 22) - h for v, h in zip((x, y), high)]
    out = np.zeros((x.shape[0], y.shape[1]), np.float32)
    chain = 128 if bits == 22 else 8192
    for k in range(0, x.shape[1], chain):
        acc = np.zeros(out.shape)
        blocks = [slice(j, min(j + 16, k + chain, x.shape[1])) for j in range(k, min(k + chain, x.shape[1]), 16)]
        if bits == 22:
            for s in blocks:
                acc = truncated(acc + high[0][:, s] @ low[1][s])
                acc = truncated(acc + low[0][:, s] @ high[1][s])
        for s in blocks:
            acc = truncated(acc + high[0][:, s] @ high[1][s])
        out += acc.astype(np.float32)
    return out.astype(np.float64)


def factor_error(u, coefficients, steps, eps, bits):
    """(factor, how far one is off whose operands are rounded to `bits` significant bits and whose sums are truncated, as a Frobenius
    norm).

    The form rounds and truncates where a kernel does: operands of every product, the completed square of a step, 23 bits of a sum.
    That way what each of the products adds is taken along through the steps that follow, which multiply it by up to their largest
    coefficient (8.2, 4 and 1.9 make 62); as one term of the result alone it is underrated by that.  A kernel's errors fall otherwise, and are of
    the same size."""
    ref = factor(u, coefficients, steps, eps)
    x = np.asarray(u, np.float64)
    x = x / max(np.sqrt(np.sum(x * x)), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    one = np.eye(len(x))
    for a, b, c in triples(coefficients, steps):
        if c == 0:
            q = a * one + b * product(x, x.T, bits)
        else:
            g = product(x, x.T, bits) + b / (2 * c) * one
            q = (a - b * b / (4 * c)) * one + c * product(g, g, bits)
        x = product(q, x, bits)
    return ref, np.linalg.norm((x.T if tall else x) - ref)
