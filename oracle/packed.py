"""Packed-sequence attention, its gradients and the relative position bias in
64 bits, with elementwise bounds on what a kernel may be off.

The bounds count roundings.  u is half a step of the 16-bit type (2^-8 bf16,
2^-11 fp16), f = 2^-24 half a step of fp32:

* a score: its product of D channels and the bias in fp32, so off by at most
  e_x = (D + 8) f (scale sum |q||k| + |bias| + |x|); e_x is at most E in a row;
* a probability: off by 2 E relative through the scores, and by 2^-16 through
  the exponential (the hardware's, 2^-22, of an argument rounded to 2^-20 where
  it counts), the row sum and its logarithm, plus n f in the sum;
* before a tensor-core product the probability (or ds) is rounded once to
  the 16-bit type: u relative, or, in fp16, half a subnormal step 2^-25 (a
  probability is held relative to its row's maximum, which is at least 1);
* a product's sum of n terms in fp32: n f of the sum of absolute terms;
* delta = dout . out takes the stored out, which is off by its own bound;
* the result is rounded once to its type.
"""
import math

import torch

F32 = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: F32}
TINY = {torch.bfloat16: 2.0 ** -125, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -125}


def bucket(rel, num_buckets, max_distance, two_sided):
    """Bucket of one key position minus query position, in whole numbers."""
    side = num_buckets // 2 if two_sided else num_buckets
    n = abs(rel) if two_sided else max(0, -rel)
    exact = side // 2
    if n < exact:
        u = n
    else:
        m, i = side - exact, 0
        while i + 1 < m and n ** m * exact ** (i + 1) >= max_distance ** (i + 1) * exact ** m:
            i += 1
        u = exact + i
    return u + (side if two_sided and rel > 0 else 0)


def bucket_matrix(nq, nk, spec, start=None):
    """[nq, nk] buckets; spec = (num_buckets, max_distance, two_sided)."""
    start = nk - nq if start is None else start
    lo, hi = -(nq - 1 + start), nk - 1 - start
    far = spec[1] + 1
    of = {}
    row = torch.tensor([of.setdefault(max(-far, min(far, r)), bucket(max(-far, min(far, r)), *spec)) for r in range(lo, hi + 1)]
                       if hi >= lo else [], dtype=torch.long)
    i = torch.arange(nq)[:, None] + start
    return row[torch.arange(nk)[None, :] - i - lo] if nq and nk else torch.zeros(nq, nk, dtype=torch.long)


def packed_attention(q, k, v, nq, nk, slots=None, causal=False, scale=None, table=None, spec=None, dout=None):
    """Values (float64) and bounds, by name: out, and with dout also grad_q,
    grad_k, grad_v, grad_table.  q [Tq, H, D], k / v [Tk, Hkv, D] as the kernel
    gets them; nq, nk, slots: lists of lengths.  Rows of no sequence are 0."""
    dev, dt = q.device, q.dtype
    u, tiny = HALF_STEP[dt], TINY[dt]
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = h // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    slots = nk if slots is None else slots
    qd, kd, vd = q.detach().double(), k.detach().double(), v.detach().double()
    td = None if table is None else table.detach().double()
    gd = None if dout is None else dout.detach().double()
    val = {"out": torch.zeros_like(qd)}
    tol = {"out": torch.zeros_like(qd)}
    if gd is not None:
        for n, t in (("grad_q", qd), ("grad_k", kd), ("grad_v", vd)) + (() if td is None else (("grad_table", td),)):
            val[n], tol[n] = torch.zeros_like(t), torch.zeros_like(t)
    q0 = k0 = 0
    for a, b, slot in zip(nq, nk, slots):
        if a and b:
            rq, rk = slice(q0, q0 + a), slice(k0, k0 + b)
            at = None if td is None else bucket_matrix(a, b, spec).to(dev)
            seen = torch.ones(a, b, dtype=torch.bool, device=dev)
            if causal:
                seen = seen.tril(b - a)
            for j in range(h):
                Q, K, V = qd[rq, j], kd[rk, j // g], vd[rk, j // g]
                x = scale * (Q @ K.t())
                mag = scale * (Q.abs() @ K.abs().t())
                if td is not None:
                    x = x + td[at, j]
                    mag = mag + td[at, j].abs()
                e = ((d + 8) * F32 * (mag + x.abs())).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                x = x.masked_fill(~seen, -math.inf)
                any_seen = seen.any(-1, keepdim=True)
                p = torch.softmax(x.masked_fill(~any_seen, 0.0), -1) * any_seen
                ep = 2 * e + 2.0 ** -16 + b * F32
                out = p @ V
                tol_out = (u + ep + b * F32) * (p @ V.abs()) + u * out.abs() + tiny * V.abs().sum(0) + tiny
                tol_out = tol_out * any_seen
                val["out"][rq, j], tol["out"][rq, j] = out, tol_out
                if gd is None:
                    continue
                DO = gd[rq, j]
                dp = DO @ V.t()
                delta = (DO * out).sum(-1, keepdim=True)
                ds = p * (dp - delta)
                e_dp = (d + 2) * F32 * (DO.abs() @ V.abs().t())
                e_delta = (DO.abs() * tol_out).sum(-1, keepdim=True) + (d + 2) * F32 * (DO * out).abs().sum(-1, keepdim=True)
                raw = ds.abs() * (ep + 4 * F32) + p * (e_dp + e_delta) * (1 + ep)  # before its rounding
                e_ds = raw + u * (ds.abs() + raw) + tiny * seen
                n = a * g
                val["grad_q"][rq, j] = scale * (ds @ K)
                tol["grad_q"][rq, j] = scale * ((e_ds + b * F32 * ds.abs()) @ K.abs()) + u * val["grad_q"][rq, j].abs() + tiny
                val["grad_k"][rk, j // g] += scale * (ds.t() @ Q)
                tol["grad_k"][rk, j // g] += scale * ((e_ds + n * F32 * ds.abs()).t() @ Q.abs())
                val["grad_v"][rk, j // g] += p.t() @ DO
                tol["grad_v"][rk, j // g] += (p * (u + ep + n * F32) + tiny * seen).t() @ DO.abs()
                if td is not None:
                    nb = td.shape[0]
                    hot = at.reshape(-1)
                    val["grad_table"][:, j].index_add_(0, hot, ds.reshape(-1))
                    tol["grad_table"][:, j].index_add_(0, hot, (raw + (a + b) * F32 * ds.abs()).reshape(-1))
                    assert nb == spec[0]
        q0, k0 = q0 + a, k0 + slot
    if gd is not None:
        for n in ("grad_k", "grad_v"):
            tol[n] += u * val[n].abs() + tiny
        if td is not None:
            tol["grad_table"] += HALF_STEP[table.dtype] * val["grad_table"].abs() + TINY[table.dtype]
    return val, tol


def relative_bias(table, queries, keys, spec, start=None):
    at = bucket_matrix(queries, keys, spec, start).to(table.device)
    return table.detach()[at].permute(2, 0, 1)


def relative_bias_grad(dbias, spec, start=None, dtype=torch.float32):
    """Value and bound of the table's gradient: an fp32 sum of n values in any
    grouping (n f of the absolute sum), rounded once to the table's type."""
    h, queries, keys = dbias.shape
    at = bucket_matrix(queries, keys, spec, start).to(dbias.device).reshape(-1)
    flat = dbias.detach().double().reshape(h, -1).t()
    val = torch.zeros(spec[0], h, dtype=torch.float64, device=dbias.device).index_add_(0, at, flat)
    mag = torch.zeros_like(val).index_add_(0, at, flat.abs())
    # the longest chain of additions: a diagonal's rows, then the diagonals
    return val, (queries + keys + 64) * F32 * mag + HALF_STEP[dtype] * val.abs() + TINY[dtype]


def packed_attention_spread(q, k, v, nq, nk, slots=None, causal=False, scale=None, table=None, spec=None, dout=None):
    """Values as packed_attention's, with bounds that add independent roundings
    by their squares: a sum of terms t, each rounded to the 16-bit type, is off
    by sqrt(sum (u t)^2 / 3) in the mean square, and by less than six times
    that in any of some millions of elements (6 / sqrt(3) = 3.5 u for a single
    term, whose rounding is at most u).  What the bounds of packed_attention
    add up in absolute value lets pass a result that is off as a whole; these
    do not.

    out: a term p v for each key.  delta = dout . out: those of out, whose error
    is sum_j r_j p_j dp_j, and out's own rounding, a term for each channel.  ds
    is rounded once a pair; delta's error is one for all pairs of a row, so it
    enters dq by |sum_j p_j k_j| and a bucket of the table by the row's sum of p
    over it.  The table's sums take ds as it is.

    fp32's errors are added in absolute value.  A score's as there.  An
    exponential is off by 2^-22 and its argument, rounded beside the row's
    maximum or logarithm (below 32 where it counts), by 2^-20; the row's sum has
    both as well: 2^-18 for all of it.  A row's sum of b terms rounds b times
    independently: 6 sqrt(b / 3) f.  The tensor cores add 16 terms a step, which
    may cut instead of round (2 f of the sum so far), and keep at least as many
    bits within the step: n terms are off by (n / 8 + 32) f.

    Below a floor a term loses all of its bits.  In fp16 a p of the gradients is
    held as 2^14 p (half a step 2^-25 - 14), and ds as 2^s ds with s from bounds
    of A = max|dout| and B = max|v| of the sequence and key head: 2^s >= 2^15 /
    (2^5.5 A B), the bounds being within sqrt(16) of A and of B and the power
    within 2^1.5, so half a step is 2^(-25 - 15 + 5.5) A B.  An exponential below
    2^-126 is 0."""
    dt = q.dtype
    u, tiny = HALF_STEP[dt], TINY[dt]
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = h // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    slots = nk if slots is None else slots
    qd, kd, vd = q.detach().double(), k.detach().double(), v.detach().double()
    td = None if table is None else table.detach().double()
    gd = None if dout is None else dout.detach().double()
    shapes = {"out": qd}
    if gd is not None:
        shapes.update(grad_q=qd, grad_k=kd, grad_v=vd)
        if td is not None:
            shapes["grad_table"] = td
    val = {n: torch.zeros_like(t) for n, t in shapes.items()}
    var = {n: torch.zeros_like(t) for n, t in shapes.items()}    # mean squares of the roundings
    slack = {n: torch.zeros_like(t) for n, t in shapes.items()}  # fp32's errors
    r2 = u * u / 3
    half = dt == torch.float16
    floor_p = 2.0 ** -39 if half else 2.0 ** -126
    q0 = k0 = 0
    for a, b, slot in zip(nq, nk, slots):
        if a and b:
            rq, rk = slice(q0, q0 + a), slice(k0, k0 + b)
            at = None if td is None else bucket_matrix(a, b, spec).to(q.device)
            seen = torch.ones(a, b, dtype=torch.bool, device=q.device)
            if causal:
                seen = seen.tril(b - a)
            any_seen = seen.any(-1, keepdim=True)
            ones = seen.double()
            for j in range(h):
                Q, K, V = qd[rq, j], kd[rk, j // g], vd[rk, j // g]
                x = scale * (Q @ K.t())
                mag = scale * (Q.abs() @ K.abs().t())
                if td is not None:
                    x, mag = x + td[at, j], mag + td[at, j].abs()
                e = ((d + 8) * F32 * (mag + x.abs())).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                x = x.masked_fill(~seen, -math.inf)
                p = torch.softmax(x.masked_fill(~any_seen, 0.0), -1) * any_seen
                ep = 2 * e + 2.0 ** -18 + 6 * math.sqrt(b / 3) * F32
                sum_b, sum_n = (b / 8 + 32) * F32, (a * g / 8 + 32) * F32
                out = p @ V
                val["out"][rq, j] = out
                var["out"][rq, j] = r2 * (p.square() @ V.square()) + (tiny * tiny * V.square().sum(0) * any_seen)
                slack["out"][rq, j] = (ep + sum_b) * (p @ V.abs())
                if gd is None:
                    continue
                DO = gd[rq, j]
                dp = DO @ V.t()
                ds = p * (dp - (DO * out).sum(-1, keepdim=True))
                # u^2 / 3 of out's own rounding, and its tiny step, a channel each
                var_delta = r2 * ((p * dp).square().sum(-1, keepdim=True) + (DO * out).square().sum(-1, keepdim=True)) + \
                    tiny * tiny * DO.square().sum(-1, keepdim=True)
                raw = ds.abs() * (ep + 4 * F32) + p * (1 + ep) * ((d + 2) * F32 * (DO.abs() @ V.abs().t())
                                                                   + ((2 * ep + (d + 2) * F32) * (DO.abs() * (p @ V.abs())).sum(-1, keepdim=True)))
                heads = slice(j // g * g, j // g * g + g)
                most = gd[rq, heads].norm(dim=-1).amax() * V.norm(dim=-1).amax()
                floor2 = (2.0 ** -34.5 * most) ** 2 if half else (2.0 ** -126 * 2 * most) ** 2
                val["grad_q"][rq, j] = scale * (ds @ K)
                var["grad_q"][rq, j] = scale ** 2 * ((r2 * ds.square() + floor2 * ones) @ K.square() + var_delta * (p @ K).square())
                slack["grad_q"][rq, j] = scale * ((raw + sum_b * ds.abs()) @ K.abs())
                val["grad_k"][rk, j // g] += scale * (ds.t() @ Q)
                var["grad_k"][rk, j // g] += scale ** 2 * ((r2 * ds.square() + floor2 * ones + var_delta * p.square()).t() @ Q.square())
                slack["grad_k"][rk, j // g] += scale * ((raw + sum_n * ds.abs()).t() @ Q.abs())
                val["grad_v"][rk, j // g] += p.t() @ DO
                var["grad_v"][rk, j // g] += (r2 * p.square() + floor_p ** 2 * ones).t() @ DO.square()
                slack["grad_v"][rk, j // g] += (p * (ep + sum_n)).t() @ DO.abs()
                if td is not None:
                    hot = at.reshape(-1)
                    val["grad_table"][:, j].index_add_(0, hot, ds.reshape(-1))
                    slack["grad_table"][:, j].index_add_(0, hot, (raw + (a + b) * F32 * ds.abs()).reshape(-1))
                    of_row = torch.zeros(a, td.shape[0], dtype=torch.float64, device=q.device).scatter_add_(1, at, p)
                    var["grad_table"][:, j] += (var_delta * of_row.square()).sum(0)
        q0, k0 = q0 + a, k0 + slot
    step = {n: HALF_STEP[table.dtype if n == "grad_table" else dt] for n in val}
    least = {n: TINY[table.dtype if n == "grad_table" else dt] for n in val}
    tol = {}
    for n in val:
        inner = 6 * var[n].sqrt() + slack[n]
        tol[n] = inner + step[n] * (val[n].abs() + inner) + least[n] * (val[n] != 0)
    return val, tol
