"""What is measured of the packed attention and of the learned relative position bias.

A case names one call of one of the two operators:

* ``prompt``: attention over whole sequences of different lengths laid one
  behind the other, forward only;
* ``train``: the same with its backward pass (the gradients of q, k, v and of
  the bias table where there is one);
* ``token``: the serving form, one (or a few) query tokens a sequence against
  a cache of fixed slots that are filled to different lengths;
* ``bias``: the bias tensor of a learned table over distance buckets, with
  the table's gradient where ``grad`` is set.

``run`` computes a case in elementary torch operations, or, where ``own`` is
set, through the framework's entry points.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def _attention(kind, name=None, **kw):
    case = dict(kind=kind, seqs=1, shortest=1, longest=1, extra_keys=0, heads=6, kv_heads=6, dim=64, dtype="bf16",
                causal=True, buckets=0, distance=0, two_sided=False, order=1)
    case.update(kw)
    if name is not None:
        case["name"] = name
    return case


def _bias(name=None, **kw):
    case = dict(kind="bias", heads=6, queries=1, keys=1, buckets=32, distance=128, two_sided=True, dtype="bf16", grad=True)
    case.update(kw)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # one user's next token against a short cache: nothing but latency
        _attention("token", "token_one_user", seqs=1, shortest=513, longest=513, heads=8, kv_heads=2, dim=64),
        # a batch of users' next tokens, caches filled to different lengths: the bytes of the cache
        _attention("token", "token_batch", seqs=64, shortest=700, longest=8192, heads=32, kv_heads=8, dim=128, order=3),
        # a few users with long caches, grouped by eight: too few rows to fill the card without splitting the keys
        _attention("token", "token_long_cache", seqs=3, shortest=30000, longest=60001, heads=16, kv_heads=2, dim=128, dtype="fp16", order=4),
        # one short prompt (an image of 14 x 14 patches and its class token)
        _attention("prompt", "prompt_one_image", seqs=1, shortest=197, longest=197, dtype="fp16", causal=False),
        # a batch of images after merging, 393 to 785 tokens left of each
        _attention("prompt", "prompt_images", seqs=128, shortest=393, longest=785, dtype="fp16", causal=False, order=5),
        # packed prompts of different lengths, grouped heads
        _attention("prompt", "prompt_packed", seqs=12, shortest=1, longest=4096, heads=16, kv_heads=4, dim=128, order=6),
        # one long prompt
        _attention("prompt", "prompt_long", seqs=1, shortest=16384, longest=16384, heads=16, kv_heads=4, dim=128),
        # a training step's attention over a batch of images, with a learned bias of their flat distance
        _attention("train", "train_images_bias", seqs=32, shortest=197, longest=785, dtype="fp16", causal=False, buckets=32, distance=128,
                   two_sided=True, order=7),
        # a training step's attention over packed documents
        _attention("train", "train_packed", seqs=7, shortest=33, longest=4000, heads=16, kv_heads=4, dim=128, order=8),
        # a training step's attention over one long document
        _attention("train", "train_long", seqs=1, shortest=8192, longest=8192, heads=16, kv_heads=8, dim=128),
        # the bias of one image's tokens, as a mask for another attention
        _bias("bias_image", queries=785, keys=785, dtype="fp16"),
        # the bias of a longer text and its gradient, one-sided
        _bias("bias_text", heads=16, queries=2048, keys=2048, buckets=32, distance=256, two_sided=False, dtype="fp32"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choice(["prompt", "train", "train", "token", "bias", "prompt"])
    if kind == "bias":
        queries = _spread(rng, 1, 2048)
        return _bias(heads=rng.choice([1, 3, 6, 8, 12, 16]), queries=queries, keys=rng.choice([queries, _spread(rng, 1, 2048)]),
                     buckets=rng.choice([16, 32, 64]), distance=rng.choice([96, 128, 256, 800]), two_sided=rng.random() < 0.5,
                     dtype=rng.choice(["bf16", "fp16", "fp32"]), grad=rng.random() < 0.7)
    heads, kv_heads = rng.choice([(6, 6), (8, 8), (8, 2), (16, 4), (12, 4), (14, 2), (16, 2), (5, 1)])
    dim = rng.choice([64, 64, 128, 128, 80, 32])
    dtype = rng.choice(["bf16", "fp16"])
    order = rng.randrange(1 << 20)
    if kind == "token":
        longest = _spread(rng, 64, 32768)
        seqs = _spread(rng, 1, max(1, min(128, 400000 // longest)))
        return _attention(kind, seqs=seqs, shortest=rng.choice([1, longest // 2 + 1]), longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                          dtype=dtype, order=order)
    most = 4.0e9 if kind == "prompt" else 1.0e9
    longest = _spread(rng, 16, 8192)
    biased = kind == "train" and longest <= 2048 and rng.random() < 0.5
    if biased:
        most /= 4
    seqs = _spread(rng, 1, max(1, min(96, int(most / (heads * longest * longest)))))
    two_sided = rng.random() < 0.5
    return _attention(kind, seqs=seqs, shortest=rng.choice([0, 1, longest // 2 + 1, longest]), longest=longest,
                      extra_keys=rng.choice([0, 0, 0, 65, -9]), heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=rng.random() < 0.7,
                      buckets=rng.choice([16, 32, 48]) if biased else 0, distance=rng.choice([64, 128, 300]) if biased else 0,
                      two_sided=two_sided if biased else False, order=order)


def _lengths(case):
    """The query and key lengths of a case's sequences, and the slots that the keys lie in."""
    rng = random.Random(case["order"])
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [hi] + [rng.randint(lo, hi) for _ in range(n - 1)]
    rng.shuffle(lens)
    if case["kind"] == "token":
        return [1] * n, lens, [hi] * n
    keys = [max(0, x + case["extra_keys"]) for x in lens]
    return lens, keys, keys


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    state = dict(case)
    if case["kind"] == "bias":
        state["table"] = (0.5 * normal(case["buckets"], case["heads"])).to(dtype).requires_grad_(case["grad"])
        state["upstream"] = normal(case["heads"], case["queries"], case["keys"]).to(dtype) if case["grad"] else None
        return state
    nq, nk, slots = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    train = case["kind"] == "train"
    state["q"] = normal(sum(nq), h, d).to(dtype).requires_grad_(train)
    state["k"] = normal(sum(slots), hk, d).to(dtype).requires_grad_(train)
    state["v"] = normal(sum(slots), hk, d).to(dtype).requires_grad_(train)
    state["dout"] = normal(sum(nq), h, d).to(dtype) if train else None
    state["table"] = (0.5 * normal(case["buckets"], h)).to(dtype).requires_grad_(train) if case["buckets"] else None
    ends = torch.tensor([0] + nq + [0] + slots, dtype=torch.int64)
    state["cu_q"] = ends[: len(nq) + 1].cumsum(0).to(torch.int32).to(DEVICE)
    state["cu_k"] = ends[len(nq) + 1:].cumsum(0).to(torch.int32).to(DEVICE)
    state["used_k"] = torch.tensor(nk, dtype=torch.int32, device=DEVICE) if case["kind"] == "token" else None
    state["max_q"], state["max_k"] = max(nq), max(nk)
    return state


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "bias":
        n = case["heads"] * case["queries"] * case["keys"]
        t = case["heads"] * case["buckets"]
        return {"bytes": size * (n + t + ((n + t) if case["grad"] else 0)), "flops": n if case["grad"] else 0}
    nq, nk, _ = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = 0
    for a, b in zip(nq, nk):
        if case["causal"]:  # query i sees keys 0 .. i + b - a
            first = max(0, b - a + 1)
            rows = a if b >= a else b
            pairs += rows * first + rows * (rows - 1) // 2 if b >= a else b * (b + 1) // 2
        else:
            pairs += a * b
    train = case["kind"] == "train"
    q, kv = sum(nq) * h * d, 2 * sum(nk) * hk * d
    return {"bytes": size * (2 * q + kv + (2 * q + kv if train else 0)) + 4 * (len(nq) + 1), "flops": (14 if train else 4) * pairs * h * d}


# ---------------------------------------------------------------- the plain forms
def _borders(case):
    """Distances at which the next bucket begins: every distance up to half of
    one side's buckets, then logarithmic up to ``distance``.  Bucket
    exact + i begins at the first whole n with
    (n / exact) ** (side - exact) >= (distance / exact) ** i, which whole
    numbers decide without rounding."""
    side = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    exact = side // 2
    m = side - exact
    found = list(range(1, exact + 1))
    n = exact
    for i in range(1, m):
        while n ** m * exact ** i < exact ** m * case["distance"] ** i:
            n += 1
        found.append(n)
    return side, found


def _bucket(case, offset):
    """The bucket of key position minus query position."""
    side, found = _borders(case)
    far = offset.abs() if case["two_sided"] else (-offset).clamp(min=0)
    at = torch.bucketize(far, torch.tensor(found, device=offset.device), right=True)
    return at + side * (offset > 0) if case["two_sided"] else at


def _plain_bias(s):
    i = torch.arange(s["queries"], device=DEVICE)[:, None] + (s["keys"] - s["queries"])
    at = _bucket(s, torch.arange(s["keys"], device=DEVICE)[None, :] - i)
    out = {"bias": s["table"].detach()[at].permute(2, 0, 1).contiguous()}
    if s["grad"]:
        up = s["upstream"].double().reshape(s["heads"], -1).t()
        grad = torch.zeros(s["buckets"], s["heads"], dtype=torch.float64, device=DEVICE).index_add_(0, at.reshape(-1), up)
        out["grad_table"] = grad.to(s["table"].dtype)
    return out


def _rows(cu, total):
    """The sequence of each packed row and its place in it."""
    r = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), r.to(torch.int32), right=True).clamp(max=cu.numel() - 2)
    return b, r - cu[b]


def _plain_attention(s):
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    g, lq, lk = h // hk, s["max_q"], s["max_k"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    n = cu_q.numel() - 1
    nq = cu_q[1:] - cu_q[:-1]
    nk = cu_k[1:] - cu_k[:-1] if s["used_k"] is None else s["used_k"].long()
    scale = 1.0 / math.sqrt(d)
    iq = torch.arange(lq, device=DEVICE)
    ik = torch.arange(lk, device=DEVICE)

    def dense(x, cu, length):  # [n, kv head, group * length, d]
        at = (cu[:-1, None] + length).clamp(max=max(0, x.shape[0] - 1))
        return x[at].reshape(n, length.numel(), hk, -1, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)

    qd, kd, vd = dense(q, cu_q, iq), dense(k, cu_k, ik), dense(v, cu_k, ik)
    offset = ik[None, None, :] - (iq[None, :, None] + (nk - nq)[:, None, None])  # [n, lq, lk]
    seen = (iq[None, :, None] < nq[:, None, None]) & (ik[None, None, :] < nk[:, None, None])
    if s["causal"]:
        seen = seen & (offset <= 0)
    scores = torch.matmul(qd, kd.transpose(-1, -2)).mul_(scale).view(n, hk, g, lq, lk)
    if s["table"] is not None:
        at = _bucket(s, offset)
        scores += s["table"].detach().float()[at].permute(0, 3, 1, 2).reshape(n, hk, g, lq, lk)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0, 1.0)).view(n, hk, g * lq, lk)
    out = torch.matmul(p, vd)
    bq, pq = _rows(cu_q, q.shape[0])

    def packed_q(x):
        return x.view(n, hk, g, lq, d).permute(0, 3, 1, 2, 4)[bq, pq].reshape(-1, h, d).to(s["q"].dtype)

    got = {"out": packed_q(out)}
    if s["kind"] != "train":
        return got
    dout = dense(s["dout"].float(), cu_q, iq) * (iq < nq[:, None]).repeat(1, g)[:, None, :, None]
    bk, pk = _rows(cu_k, k.shape[0])

    def packed_k(x):
        return (x.permute(0, 2, 1, 3)[bk, pk] * (pk < nk[bk])[:, None, None]).to(s["k"].dtype)

    got["grad_v"] = packed_k(torch.matmul(p.transpose(-1, -2), dout))
    dp = torch.matmul(dout, vd.transpose(-1, -2))
    ds = dp.sub_((dout * out).sum(-1, keepdim=True)).mul_(p)
    got["grad_q"] = packed_q(torch.matmul(ds, kd) * scale)
    got["grad_k"] = packed_k(torch.matmul(ds.transpose(-1, -2), qd) * scale)
    if s["table"] is not None:
        each = ds.view(n, h, lq, lk).permute(0, 2, 3, 1).reshape(-1, h).double()
        grad = torch.zeros(s["buckets"], h, dtype=torch.float64, device=DEVICE).index_add_(0, at.reshape(-1), each)
        got["grad_table"] = grad.to(s["table"].dtype)
    return got


# ------------------------------------------------------- the framework's entry points
def _own(s):
    import mergenet_b200 as mn

    buckets = None
    if s["buckets"]:
        buckets = mn.RelativeBuckets(s["buckets"], s["distance"], s["two_sided"])
    if s["kind"] == "bias":
        bias = mn.relative_position_bias(s["table"], s["queries"], s["keys"], buckets)
        if not s["grad"]:
            return {"bias": bias}
        return {"bias": bias.detach(), "grad_table": torch.autograd.grad(bias, s["table"], s["upstream"])[0]}
    out = mn.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], lengths_k=s["used_k"], causal=s["causal"], bias_table=s["table"],
                              buckets=buckets)
    if s["kind"] != "train":
        return {"out": out}
    leaves = [s["q"], s["k"], s["v"]] + ([] if s["table"] is None else [s["table"]])
    grads = torch.autograd.grad(out, leaves, s["dout"])
    return dict(zip(["out", "grad_q", "grad_k", "grad_v", "grad_table"], [out.detach(), *grads]))


def run(state):
    if own:
        return _own(state)
    return _plain_bias(state) if state["kind"] == "bias" else _plain_attention(state)


# ------------------------------------------------------------------- in 64 bits
def _side_of(case, n):
    """The bucket of a distance n >= 0 on one side, from the formula
    exact + floor(log(n / exact) / log(distance / exact) * m), its logarithms
    raised to whole powers so that nothing is rounded."""
    side = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    exact = side // 2
    if n < exact:
        return n
    m, i = side - exact, 0
    while i + 1 < m and n ** m * exact ** (i + 1) >= case["distance"] ** (i + 1) * exact ** m:
        i += 1
    return exact + i


def _exact_buckets(case, nq, nk):
    half = case["buckets"] // 2
    of = []
    for rel in range(-(nk + nq), nk + nq + 1):
        n = min(abs(rel) if case["two_sided"] else max(0, -rel), 2 * case["distance"])
        of.append(_side_of(case, n) + (half if case["two_sided"] and rel > 0 else 0))
    i = torch.arange(nq)[:, None] + nk - nq
    return torch.tensor(of)[torch.arange(nk)[None, :] - i + nk + nq].to(DEVICE)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "bias":
        at = _exact_buckets(case, case["queries"], case["keys"])
        table = s["table"].detach().double().requires_grad_(case["grad"])
        bias = torch.stack([table[:, j][at] for j in range(case["heads"])])
        if not case["grad"]:
            return {"bias": bias}
        return {"bias": bias.detach(), "grad_table": torch.autograd.grad(bias, table, s["upstream"].double())[0]}
    nq, nk, slots = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    g, train = h // hk, case["kind"] == "train"
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    table = None if s["table"] is None else s["table"].detach().double()
    out, gq, gk, gv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    gt = None if table is None else torch.zeros_like(table)
    q0 = k0 = 0
    for a, b, slot in zip(nq, nk, slots):
        if a and b:
            at = None if table is None else _exact_buckets(case, a, b)
            hidden = torch.ones(a, b, dtype=torch.bool, device=DEVICE).triu(b - a + 1) if case["causal"] else None
            for j in range(h):
                mine = [q[q0:q0 + a, j], k[k0:k0 + b, j // g], v[k0:k0 + b, j // g]] + ([] if table is None else [table[:, j]])
                mine = [x.clone().requires_grad_(train) for x in mine]
                x = mine[0] @ mine[1].t() / math.sqrt(d)
                if table is not None:
                    x = x + mine[3][at]
                if hidden is not None:
                    x = x.masked_fill(hidden, -math.inf)
                    none = hidden.all(-1, keepdim=True)
                    p = torch.softmax(x.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
                else:
                    p = torch.softmax(x, -1)
                o = p @ mine[2]
                out[q0:q0 + a, j] = o.detach()
                if train:
                    grads = torch.autograd.grad(o, mine, s["dout"][q0:q0 + a, j].double())
                    gq[q0:q0 + a, j] = grads[0]
                    gk[k0:k0 + b, j // g] += grads[1]
                    gv[k0:k0 + b, j // g] += grads[2]
                    if table is not None:
                        gt[:, j] += grads[3]
                del x, p, o
        q0, k0 = q0 + a, k0 + slot
    if not train:
        return {"out": out}
    got = {"out": out, "grad_q": gq, "grad_k": gk, "grad_v": gv}
    if gt is not None:
        got["grad_table"] = gt
    return got
