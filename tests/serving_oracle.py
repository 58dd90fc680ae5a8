"""Plain 64-bit implementations of the serving operators on the CPU, and the bounds their tests hold the kernels to."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}


def attention(q, k, v, visible, divisor, cap=0.0, bias=None):
    """q [n, d], k, v [m, d], visible [n, m] -> (context, sum of |weight * value|), rows that see nothing zero.  What a query
    does not see is taken out before the products, so it may hold anything."""
    q, k, v = q.double(), k.double(), v.double()
    out, size = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64), torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    for i in range(q.shape[0]):
        seen = visible[i].nonzero()[:, 0]
        if len(seen) == 0:
            continue
        s = k[seen] @ q[i] / divisor
        if cap:
            s = cap * torch.tanh(s / cap)
        if bias is not None:
            s = s + bias[i, seen]
        p = torch.softmax(s, 0)
        out[i], size[i] = p @ v[seen], p @ v[seen].abs()
    return out, size


def bound(dtype, size, out):
    """How far a context may be off, element by element.

    A weight: half a step of the type where it is rounded for the second product (16-bit types), and the score's error twice
    (numerator and sum).  A score of values ~ N(0, 1) and head size up to 128 sums |q||k| / divisor of about 7 (up to three times
    that here): the sums of a tensor core lose at most 2^-23 of the running size per instruction of 16 (8) products, which is
    8 x 2^-23 x 21 = 2e-5 for 16-bit types and, in TF32 triples (48 instructions) with 2^-21 lost to the split of either
    operand, (48 x 2^-23 + 2^-20) x 21 = 1.4e-4 for fp32; the exponential's 2^-22 and the capped score's 1e-7 x cap stay below
    1e-5.  The context's own sum adds 2^-23 per instruction, below 1e-5 for the lengths here.  The result is rounded once."""
    step = HALF_STEP[dtype]
    weight = 3e-4 if dtype == torch.float32 else step + 1e-4
    return weight * size + step * out.abs() + 1e-7


def close(got, want, size, dtype):
    err = (got.double().cpu() - want).abs()
    return bool((err <= bound(dtype, size, want)).all())


def sample(logits, u, temperature, top_k, top_p, min_p):
    """(token, probability, distance) of one row; distance: how near the draw or a cut is to the next outcome, in weights of
    the largest.  Python floats throughout, math.fsum for the sums."""
    z = [float(x) for x in logits]
    z = [-math.inf if x != x else x for x in z]
    top = max(z)
    if top == -math.inf:
        return -1, 0.0, 1.0
    order = sorted(range(len(z)), key=lambda i: (-z[i], i))
    if not temperature > 0:
        return order[0], 1.0, 1.0
    temperature = max(temperature, 1e-30)

    def weight(x):
        if x == top:
            return 1.0
        return 0.0 if top == math.inf or x == -math.inf else math.exp((x - top) / temperature)

    order = [i for i in order if z[i] > -math.inf]
    if 0 < top_k < len(order):
        order = order[:top_k]
    w = [weight(z[i]) for i in order]
    near = 1.0
    if top_p < 1:
        want = max(top_p, 0.0) * math.fsum(w)
        before, n = 0.0, 0
        while n < len(w) and (n == 0 or before < want):
            before = math.fsum(w[:n + 1])
            near = min(near, abs(before - want)) if want else near
            n += 1
        order, w = order[:n], w[:n]
    if min_p > 0:
        kept = [x >= min(min_p, 1.0) for x in w]
        near = min([near] + [abs(x - min_p) for x in w if x != 1.0])
        order, w = [i for i, s in zip(order, kept) if s], [x for x, s in zip(w, kept) if s]
    back = sorted(range(len(order)), key=lambda j: order[j])
    total = math.fsum(w)
    u = min(max(u, 0.0), 0.99999994) if u == u else 0.0
    run, token, at = 0.0, None, 0.0
    for n, j in enumerate(back):
        run += w[j]
        near = min(near, abs(run - u * total))
        if token is None and run > u * total:
            token, at = order[j], w[j]
    return token, at / total, near
