"""The packed attention, its gradients and the relative position bias on the
GPU against the 64-bit oracle, within the bounds that the oracle derives from
the roundings of the path."""
import pytest
import torch

from oracle import packed as O

pytestmark = pytest.mark.gpu

SPEC = (32, 128, True)


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import mergenet_b200  # noqa: F401
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _status_stays_clear():
    import mergenet_b200
    d = torch.device("cuda", 0)
    mergenet_b200.attention.attention_status(d, reset=True)
    yield
    assert mergenet_b200.attention.attention_status(d, reset=True) == 0


def offsets(lens, dev):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(dev)


def randn(gen, *shape, dtype=torch.bfloat16, amp=1.0):
    return (amp * torch.randn(*shape, generator=gen, device=gen.device)).to(dtype)


def problem(dev, nq, nk=None, slots=None, heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16, spec=None, seed=0, extra=0,
            table_dtype=None):
    gen = torch.Generator(device=dev).manual_seed(seed)
    nk = nq if nk is None else nk
    slots = nk if slots is None else slots
    p = dict(q=randn(gen, sum(nq) + extra, heads, dim, dtype=dtype), k=randn(gen, sum(slots) + extra, kv_heads, dim, dtype=dtype),
             v=randn(gen, sum(slots) + extra, kv_heads, dim, dtype=dtype))
    p["table"] = randn(gen, spec[0], heads, dtype=table_dtype or dtype) if spec else None
    p["dout"] = randn(gen, sum(nq) + extra, heads, dim, dtype=dtype)
    p.update(nq=nq, nk=nk, slots=slots, spec=spec)
    return p


def call(p, causal, grads, scale=None, lengths=None):
    import mergenet_b200 as mn
    dev = p["q"].device
    buckets = mn.RelativeBuckets(*p["spec"]) if p["spec"] else None
    leaves = {"grad_" + n: p[n].detach().requires_grad_(grads) for n in ("q", "k", "v", "table") if p[n] is not None}
    out = mn.packed_attention(leaves["grad_q"], leaves["grad_k"], leaves["grad_v"], offsets(p["nq"], dev), offsets(p["slots"], dev),
                              lengths_k=lengths, causal=causal, scale=scale, bias_table=leaves.get("grad_table"), buckets=buckets)
    got = {"out": out.detach()}
    if grads:
        got.update(zip(leaves, torch.autograd.grad(out, list(leaves.values()), p["dout"])))
    return got


def check(got, p, causal, scale=None):
    val, tol = O.packed_attention(p["q"], p["k"], p["v"], p["nq"], p["nk"], p["slots"], causal=causal, scale=scale, table=p["table"],
                                  spec=p["spec"], dout=p["dout"] if "grad_q" in got else None)
    for name, x in got.items():
        assert torch.isfinite(x.float()).all(), name
        if not x.numel():
            continue
        off = (x.double() - val[name]).abs()
        worst = float((off - tol[name]).max())
        assert worst <= 0, f"{name}: {float(off.max()):.3e} off, past its bound by {worst:.3e}"


LENGTHS = {
    "one": ([1], None),
    "empty_between": ([1, 0, 5, 33], None),
    "tile_edges": ([127, 128, 129, 64, 65], None),
    "two_tiles": ([256, 257, 300], None),
    "images": ([393, 785, 197], None),
    "more_queries": ([70, 130, 9], [33, 2, 0]),
    "more_keys": ([3, 64, 130], [300, 65, 513]),
    "no_keys_at_all": ([5, 3], [0, 0]),
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_lengths(dev, lengths, causal):
    nq, nk = LENGTHS[lengths]
    p = problem(dev, nq, nk)
    check(call(p, causal, True), p, causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 6, 64), (8, 2, 128), (16, 2, 64), (6, 2, 128), (7, 1, 80), (5, 1, 8), (3, 3, 96),
                                               (2, 1, 32), (32, 1, 16), (130, 2, 8)])
def test_heads_and_widths(dev, heads, kv_heads, dim, dtype):
    p = problem(dev, [150, 1, 40], [150, 77, 200], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    check(call(p, True, True), p, True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spec", [(32, 128, True), (32, 128, False), (16, 40, True), (48, 700, False), (4, 2, True)])
@pytest.mark.parametrize("causal", [False, True])
def test_bias(dev, spec, causal, dtype):
    p = problem(dev, [300, 1, 129], [300, 290, 64], dtype=dtype, spec=spec, heads=4, kv_heads=2)
    check(call(p, causal, True), p, causal)


@pytest.mark.parametrize("heads,kv_heads,dim,table_dtype", [(32, 2, 64, torch.float16), (16, 1, 128, torch.float16), (12, 4, 80, torch.float32),
                                                            (6, 6, 64, torch.float32), (8, 1, 128, torch.bfloat16),
                                                            (5, 1, 128, torch.float32), (14, 2, 64, torch.float16)])
def test_bias_heads(dev, heads, kv_heads, dim, table_dtype):
    p = problem(dev, [200, 520], heads=heads, kv_heads=kv_heads, dim=dim, spec=SPEC, table_dtype=table_dtype)
    check(call(p, False, True), p, False)


@pytest.mark.parametrize("kv_lengths", [[1], [128, 1, 257, 4000], [0, 5, 900]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (32, 8, 128), (6, 6, 64)])
def test_single_tokens(dev, kv_lengths, heads, kv_heads, dim):
    p = problem(dev, [1] * len(kv_lengths), kv_lengths, heads=heads, kv_heads=kv_heads, dim=dim)
    check(call(p, True, False), p, True)
    check(call(p, True, True), p, True)


def test_long_cache_is_split_and_joined(dev):
    p = problem(dev, [1, 2, 1], [30001, 12345, 7], heads=8, kv_heads=2, dim=128, dtype=torch.float16)
    check(call(p, True, False), p, True)


def test_single_token_with_bias(dev):
    p = problem(dev, [1, 1, 3], [700, 9, 1300], spec=(32, 256, False), heads=8, kv_heads=2)
    check(call(p, True, False), p, True)


def test_long_sequence(dev):
    p = problem(dev, [2500], heads=4, kv_heads=1, dim=128)
    check(call(p, True, True), p, True)


def test_cache_past_32_bit_offsets(dev):
    """A cache of more than 2^31 values, the sequences at its end; only their
    rows are ever written."""
    import mergenet_b200 as mn
    rows, hk, d = (1 << 21) + 700, 8, 128
    k = torch.empty(rows, hk, d, device=dev, dtype=torch.bfloat16)
    v = torch.empty(rows, hk, d, device=dev, dtype=torch.bfloat16)
    assert k.numel() > 1 << 31
    p = problem(dev, [3, 1], [300, 400], heads=16, kv_heads=hk, dim=d)
    k[-700:], v[-700:] = p["k"], p["v"]
    cu_k = torch.tensor([0, rows - 700, rows - 400, rows], dtype=torch.int32, device=dev)
    cu_q = torch.tensor([0, 0, 3, 4], dtype=torch.int32, device=dev)
    leaves = [t.detach().requires_grad_(True) for t in (p["q"], k, v)]
    out = mn.packed_attention(*leaves, cu_q, cu_k, causal=True)
    gq, gk, gv = torch.autograd.grad(out, leaves, p["dout"])
    check({"out": out.detach(), "grad_q": gq, "grad_k": gk[-700:], "grad_v": gv[-700:]}, p, True)
    assert not gk[:4096].any() and not gk[-4796:-700].any() and not gv[-4796:-700].any()


def test_two_streams_at_once(dev):
    """The same call on two streams at the same time: nothing is shared."""
    p = [problem(dev, [1] * 4, [9000, 50, 4000, 700], heads=8, kv_heads=2, dim=128, seed=s) for s in (1, 2)]
    t = [problem(dev, [300, 129], spec=SPEC, seed=s) for s in (3, 4)]
    want = [call(x, True, False) for x in p], [call(x, True, True) for x in t]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[0][i].append(call(p[i], True, False))
                got[1][i].append(call(t[i], True, True))
    torch.cuda.synchronize()
    for kind in range(2):
        for i in range(2):
            for g in got[kind][i]:
                for n in g:
                    assert torch.equal(g[n], want[kind][i][n]), n


def test_split_calls_in_captured_graphs(dev):
    """Two graphs of a call that divides its keys, replayed in turn: each has
    its own workspace."""
    import mergenet_b200 as mn
    p = [problem(dev, [1, 1], [20000, 3000], heads=8, kv_heads=2, dim=128, seed=s) for s in (1, 2)]
    want = [call(x, True, False)["out"] for x in p]
    cu_q, cu_k = offsets([1, 1], dev), offsets([20000, 3000], dev)
    graphs = []
    for x in p:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mn.packed_attention(x["q"], x["k"], x["v"], cu_q, cu_k, causal=True)
        graphs.append((graph, out))
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], want[i])


def test_leaf_used_twice(dev):
    """k and v the same tensor: its gradient is the sum of both."""
    import mergenet_b200 as mn
    p = problem(dev, [140, 30], heads=4, kv_heads=2, dtype=torch.float16)
    p["v"] = p["k"]
    kv = p["k"].detach().requires_grad_(True)
    q = p["q"].detach().requires_grad_(True)
    out = mn.packed_attention(q, kv, kv, offsets(p["nq"], dev), causal=True)
    gq, gkv = torch.autograd.grad(out, [q, kv], p["dout"])
    val, tol = O.packed_attention(p["q"], p["k"], p["v"], p["nq"], p["nk"], causal=True, dout=p["dout"])
    total = val["grad_k"] + val["grad_v"]
    # both gradients are within their bounds, and their sum is rounded once more
    bound = tol["grad_k"] + tol["grad_v"]
    assert bool(((gkv.double() - total).abs() <= bound + 2.0 ** -11 * (total.abs() + bound)).all())
    assert bool(((gq.double() - val["grad_q"]).abs() <= tol["grad_q"]).all())


def test_many_sequences(dev):
    g = torch.Generator().manual_seed(3)
    nq = torch.randint(0, 40, (300,), generator=g).tolist()
    nk = torch.randint(0, 60, (300,), generator=g).tolist()
    p = problem(dev, nq, nk, heads=2, kv_heads=1)
    check(call(p, True, True), p, True)


def test_more_sequences_than_one_tile_walk(dev):
    nq = [1] * 5000
    p = problem(dev, nq, heads=2, kv_heads=2)
    got = call(p, False, True)
    # one key each: the output is v, every score gradient is 0
    assert torch.equal(got["out"], p["v"])
    assert torch.equal(got["grad_v"], p["dout"])


@pytest.mark.parametrize("amp", [8.0, 30.0])
def test_large_scores(dev, amp):
    p = problem(dev, [200, 90], dtype=torch.bfloat16)
    p["q"] = (p["q"].float() * amp).bfloat16()
    check(call(p, True, True), p, True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** -3, 1.0, 64.0])
def test_scores_past_the_integers_of_fp32(dev, scale, dtype):
    """Scores of 10^7 to 10^10 that fp32 no longer resolves to 1: rows whose
    best key leads by more than the scores' error take that key alone.  The
    others stay finite."""
    p = problem(dev, [300, 1, 150], dtype=dtype, heads=4, kv_heads=2)
    p["q"], p["k"] = p["q"] * 4000, p["k"] * 4000
    got = call(p, True, True, scale=scale)
    for n, x in got.items():
        if n in ("out", "grad_v"):  # dq and dk have factors of 4000 x scale, past fp16's range
            assert torch.isfinite(x.float()).all(), n
    sure = 0
    r0 = 0
    for n in p["nq"]:
        rows = slice(r0, r0 + n)
        for h in range(4):
            q, k = p["q"][rows, h].double(), p["k"][rows, h // 2].double()
            off = (64 + 8) * O.F32 * 2 * scale * (q.abs() @ k.abs().t()).amax(-1)
            x = (scale * (q @ k.t())).masked_fill(~torch.ones(n, n, dtype=torch.bool, device=dev).tril(), -float("inf"))
            top = x.topk(min(2, n), dim=-1)
            lead = top.values[:, 0] - top.values[:, 1] if n > 1 else torch.full((n,), float("inf"), device=dev)
            clear = lead > 2 * off + 200  # e^-200 is 0 in fp32
            assert torch.equal(got["out"][rows, h][clear], p["v"][rows, h // 2][top.indices[:, 0]][clear])
            sure += int(clear.sum())
        r0 += n
    assert sure > 900  # of 1,804 rows


HIDDEN = [-1e4, -65504.0, -1e9, -1e30, torch.finfo(torch.float32).min, -float("inf")]


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_a_table_that_hides_distances(dev, hidden, dtype, dim):
    """The outermost buckets at a mask's value: keys that far away have no
    weight, whichever value it is.  The oracle hides them by -200, whose
    e^-200 lies below every bound, so that the bounds stay those of the rest."""
    p = problem(dev, [700, 1, 129], [700, 640, 129], dtype=dtype, dim=dim, spec=SPEC, table_dtype=torch.float32)
    table = p["table"].clone()
    for bucket in (15, 31):
        p["table"][bucket] = -200.0
        table[bucket] = hidden
    for causal in (False, True):
        got = call(dict(p, table=table), causal, True)
        check(got, p, causal)
        assert not got["grad_table"][[15, 31]].any()


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_rows_that_a_table_hides_whole(dev, hidden, dtype, dim):
    """Queries ahead of all keys, whose buckets are all hidden.  A finite value
    is the same for all of them and leaves the softmax of the scores (fp32
    keeps a little of them beside a large value); -inf leaves nothing."""
    p = problem(dev, [200], [50], dtype=dtype, dim=dim, spec=SPEC, table_dtype=torch.float32)
    p["table"][16:] = 0.0
    table = p["table"].clone()
    table[16:] = hidden
    ahead = 200 - 50  # rows of positions below 0
    got = call(dict(p, table=table), False, True)
    for n, x in got.items():
        assert torch.isfinite(x.float()).all(), n
    if hidden == -float("inf"):
        assert not got["out"][:ahead].any() and not got["grad_q"][:ahead].any()
        assert not got["grad_table"][16:].any()
    else:  # weights of the keys within a factor: each output a mean of the values
        val, tol = O.packed_attention(p["q"], p["k"], p["v"], p["nq"], p["nk"], table=p["table"], spec=p["spec"])
        # beside 2^17 the sum of a score and the hidden value is off by 2^-7 at
        # most, in log2 units, and so is the row's logarithm
        slack = 4 * 2.0 ** -7 * p["v"].double().abs().amax()
        assert ((got["out"].double() - val["out"]).abs()[:ahead] <= tol["out"][:ahead] + slack).all()


def test_growing_maxima(dev):
    """Scores that grow along the keys by far more than one rescale step."""
    p = problem(dev, [600], heads=2, kv_heads=2, dtype=torch.float16)
    ramp = torch.linspace(0.1, 6.0, 600, device=dev)[:, None, None]
    p["k"] = (p["q"].float().sign() * ramp).half()
    check(call(p, False, True), p, False)
    p["k"] = p["k"].flip(0)
    check(call(p, False, True), p, False)


def test_scale(dev):
    p = problem(dev, [130, 20])
    check(call(p, True, True, scale=0.02), p, True, scale=0.02)


def test_views_of_a_packed_projection_and_head_major_layout(dev):
    import mergenet_b200 as mn
    gen = torch.Generator(device=dev).manual_seed(1)
    nq = [100, 37, 140]
    qkv = randn(gen, sum(nq), (4 + 2 + 2) * 64)
    q, k, v = qkv.view(sum(nq), 8, 64).split([4, 2, 2], 1)
    want = mn.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets(nq, dev), causal=True)
    assert torch.equal(mn.packed_attention(q, k, v, offsets(nq, dev), causal=True), want)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(mn.packed_attention(*hm, offsets(nq, dev), causal=True), want)
    odd = [torch.empty(sum(nq), t.shape[1], 65, device=dev, dtype=t.dtype)[..., :64].copy_(t) for t in (q, k, v)]
    assert torch.equal(mn.packed_attention(*odd, offsets(nq, dev), causal=True), want)
    shifted = torch.empty(qkv.numel() + 1, device=dev, dtype=qkv.dtype)[1:].view_as(qkv).copy_(qkv)
    sq, sk, sv = shifted.view(sum(nq), 8, 64).split([4, 2, 2], 1)
    assert torch.equal(mn.packed_attention(sq, sk, sv, offsets(nq, dev), causal=True), want)
    # one row of keys for every position (stride 0), and a broadcast gradient
    k1 = k[:1].expand(sum(nq), -1, -1)
    assert torch.equal(mn.packed_attention(q, k1, v, offsets(nq, dev)), mn.packed_attention(q, k1.contiguous(), v, offsets(nq, dev)))
    lq = q.detach().clone().requires_grad_(True)
    mn.packed_attention(lq, k, v, offsets(nq, dev), causal=True).float().sum().backward()
    l2 = q.detach().clone().requires_grad_(True)
    out = mn.packed_attention(l2, k, v, offsets(nq, dev), causal=True)
    out.backward(torch.ones_like(out))
    assert torch.equal(lq.grad, l2.grad)


def test_gradients_through_a_packed_projection(dev):
    """The gradient of a projection whose views are q, k and v."""
    import mergenet_b200 as mn
    p = problem(dev, [90, 41], heads=4, kv_heads=4)
    qkv = torch.cat([p["q"], p["k"], p["v"]], 1).detach().requires_grad_(True)
    q, k, v = qkv.split(4, 1)
    out = mn.packed_attention(q, k, v, offsets(p["nq"], dev), causal=True)
    out.backward(p["dout"])
    got = dict(zip(["grad_q", "grad_k", "grad_v"], qkv.grad.split(4, 1)))
    check({"out": out.detach(), **got}, p, True)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_outside_the_sequences_reach_nothing(dev, poison, dim):
    """Unused cache rows and rows behind the last sequence hold NaN or
    infinities: results are those of clean rows, and their gradients are 0."""
    nq, nk, slots = [70, 1, 130, 0], [70, 100, 130, 3], [200, 128, 256, 5]
    p = problem(dev, nq, nk, slots, dim=dim, extra=77)
    used = torch.zeros(sum(slots) + 77, dtype=torch.bool, device=dev)
    k0 = 0
    for b, s in zip(nk, slots):
        used[k0:k0 + b] = True
        k0 += s
    lens = torch.tensor(nk, dtype=torch.int32, device=dev)
    clean = call(p, True, True, lengths=lens)
    check({n: x for n, x in clean.items()}, p, True)
    p["k"][~used] = poison
    p["v"][~used] = poison
    p["q"][sum(nq):] = poison
    p["dout"][sum(nq):] = poison
    got = call(p, True, True, lengths=lens)
    for name in clean:
        assert torch.equal(got[name], clean[name]), name
    assert not got["out"][sum(nq):].any() and not got["grad_q"][sum(nq):].any()
    assert not got["grad_k"][~used].any() and not got["grad_v"][~used].any()


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_other_sequences_reach_nothing(dev, poison, dim):
    nq = [70, 50, 131]
    p = problem(dev, nq, dim=dim, spec=SPEC)
    clean = call(p, False, True)
    for n in ("q", "k", "v", "dout"):
        p[n][70:120] = poison
    got = call(p, False, True)
    rest = torch.cat([torch.arange(70), torch.arange(120, 251)]).to(dev)
    for name in ("out", "grad_q", "grad_k", "grad_v"):
        assert torch.equal(got[name][rest], clean[name][rest]), name


def test_a_nan_score_shows(dev):
    p = problem(dev, [40, 30])
    p["q"][3, 1] = float("nan")
    got = call(p, False, False)["out"]
    assert torch.isnan(got[3, 1]).all()
    got[3, 1] = 0
    assert torch.isfinite(got).all()


def test_equal_calls_give_equal_bits(dev):
    p = problem(dev, [500, 3, 260], heads=8, kv_heads=2, dim=128, spec=SPEC)
    a = call(p, True, True)
    for _ in range(3):
        b = call(p, True, True)
        for n in a:
            assert torch.equal(a[n], b[n]), n


def test_bad_offsets_set_the_status(dev):
    """Offsets past the end and decreasing: in-bounds, and reported."""
    import mergenet_b200 as mn
    from mergenet_b200 import _lib as L
    p = problem(dev, [30, 40])
    for bad in ([0, 30, 900], [0, 50, 20], [-4, 30, 70], [0, 2 ** 31 - 1, -2 ** 31]):
        cu = torch.tensor(bad, dtype=torch.int32, device=dev)
        leaf = p["q"].detach().requires_grad_(True)
        mn.packed_attention(leaf, p["k"], p["v"], cu, causal=True).sum().backward()
        assert mn.attention.attention_status(dev, reset=True) & L.MN_STATUS_BAD_LENGTHS
    lens = torch.tensor([31, -1], dtype=torch.int32, device=dev)
    mn.packed_attention(p["q"], p["k"], p["v"], offsets(p["nq"], dev), lengths_k=lens)
    assert mn.attention.attention_status(dev, reset=True) & L.MN_STATUS_BAD_LENGTHS


@pytest.mark.parametrize("tq,tk", [(0, 0), (0, 5), (5, 0)])
def test_empty_tensors(dev, tq, tk):
    p = problem(dev, [tq], [tk], spec=SPEC)
    got = call(p, False, True)
    for n, x in got.items():
        assert not x.any(), n
    assert got["out"].shape == (tq, 4, 64) and got["grad_k"].shape == (tk, 2, 64)


def test_side_stream_and_captured_calls(dev):
    """A training call on another stream, and two captured graphs replayed in
    turn on new inputs, against eager calls."""
    import mergenet_b200 as mn
    p = [problem(dev, [150, 60], heads=4, kv_heads=2, spec=SPEC, seed=s) for s in (1, 2)]
    want = [call(x, True, True) for x in p]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(p[0], True, True)
    torch.cuda.current_stream().wait_stream(side)
    for n in got:
        assert torch.equal(got[n], want[0][n]), n
    buckets, cu = mn.RelativeBuckets(*SPEC), offsets([150, 60], dev)
    graphs = []
    for i in range(2):
        still = {n: p[0][n].detach().clone() for n in ("q", "k", "v", "table", "dout")}
        for n in ("q", "k", "v", "table"):
            still[n].requires_grad_(True)
        leaves = [still[n] for n in ("q", "k", "v", "table")]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mn.packed_attention(*leaves[:3], cu, causal=True, bias_table=leaves[3], buckets=buckets)
            grads = torch.autograd.grad(out, leaves, still["dout"])
        graphs.append((graph, still, [out.detach(), *grads]))
    for order in ((0, 1), (1, 0)):
        for i in order:  # each graph gets the problem of its place in the order
            with torch.no_grad():
                for n in ("q", "k", "v", "table", "dout"):
                    graphs[i][1][n].copy_(p[order.index(i)][n])
        for i in order:
            graphs[i][0].replay()
        for i in order:
            for x, n in zip(graphs[i][2], want[0]):
                assert torch.equal(x, want[order.index(i)][n]), n


def test_double_backward_is_refused(dev):
    p = problem(dev, [20])
    q = p["q"].detach().requires_grad_(True)
    import mergenet_b200 as mn
    out = mn.packed_attention(q, p["k"], p["v"], offsets([20], dev))
    (g,) = torch.autograd.grad(out, q, torch.ones_like(out).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ------------------------------------------------------- the bias as a tensor
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,queries,keys,start", [(1, 1, 1, None), (6, 197, 197, None), (3, 1, 700, None), (5, 130, 67, None),
                                                      (2, 65, 300, 4), (4, 64, 64, -90), (2, 33, 1027, 5000), (16, 785, 785, None),
                                                      (3, 1027, 8, None)])
@pytest.mark.parametrize("spec", [(32, 128, True), (16, 40, False), (64, 800, False)])
def test_relative_bias(dev, dtype, heads, queries, keys, start, spec):
    import mergenet_b200 as mn
    gen = torch.Generator(device=dev).manual_seed(queries)
    table = randn(gen, spec[0], heads, dtype=dtype).requires_grad_(True)
    up = randn(gen, heads, queries, keys, dtype=dtype)
    bias = mn.relative_position_bias(table, queries, keys, mn.RelativeBuckets(*spec), query_start=start)
    assert bias.dtype == dtype and torch.equal(bias.detach(), O.relative_bias(table, queries, keys, spec, start))
    (grad,) = torch.autograd.grad(bias, table, up)
    val, tol = O.relative_bias_grad(up, spec, start, dtype)
    assert grad.dtype == dtype and bool(((grad.double() - val).abs() <= tol).all())


def test_relative_bias_layouts_and_empty(dev):
    import mergenet_b200 as mn
    b = mn.RelativeBuckets(*SPEC)
    gen = torch.Generator(device=dev).manual_seed(0)
    wide = randn(gen, 32, 9, dtype=torch.float32)
    assert torch.equal(mn.relative_position_bias(wide[:, 2:5], 40, 50, b), mn.relative_position_bias(wide[:, 2:5].contiguous(), 40, 50, b))
    table = randn(gen, 32, 3, dtype=torch.float32).requires_grad_(True)
    mn.relative_position_bias(table, 40, 50, b).sum().backward()  # a broadcast gradient
    val, tol = O.relative_bias_grad(torch.ones(3, 40, 50, device=dev), SPEC)
    assert bool(((table.grad.double() - val).abs() <= tol).all())
    for shape in ((0, 5), (5, 0)):
        bias = mn.relative_position_bias(table, *shape, b)
        assert bias.shape == (3, *shape)
        assert not torch.autograd.grad(bias, table, torch.zeros_like(bias))[0].any()


def test_both_together_in_a_training_step(dev):
    """The bias inside the attention and the bias as a tensor are the same
    operator: one step of a layer that uses the table in both ways gets the
    sum of both gradients, and the attention agrees with plain products over
    the bias tensor."""
    import mergenet_b200 as mn
    p = problem(dev, [120, 75], heads=4, kv_heads=4, spec=SPEC, dtype=torch.float16)
    buckets = mn.RelativeBuckets(*SPEC)
    table = p["table"].detach().float().requires_grad_(True)
    q, k, v = (p[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    out = mn.packed_attention(q, k, v, offsets(p["nq"], dev), bias_table=table, buckets=buckets)
    bias = mn.relative_position_bias(table, 120, 120, buckets)
    x = torch.einsum("ihd,jhd->hij", q.detach()[:120].double(), k.detach()[:120].double()) / 8 + bias.detach().double()
    plain = torch.einsum("hij,jhd->ihd", torch.softmax(x, -1), v.detach()[:120].double())
    ((out.float() * p["dout"].float()).sum() + bias.square().sum()).backward()
    p["table"] = table.detach()
    val, tol = O.packed_attention(p["q"], p["k"], p["v"], p["nq"], p["nk"], table=p["table"], spec=SPEC, dout=p["dout"])
    assert bool(((out.detach().double() - val["out"]).abs() <= tol["out"]).all())
    assert bool(((plain - val["out"][:120]).abs() <= tol["out"][:120]).all())
    more, more_tol = O.relative_bias_grad(2 * bias.detach(), SPEC)
    total = val["grad_table"] + more
    # each gradient is rounded to fp32, and their sum again
    assert bool(((table.grad.double() - total).abs() <= tol["grad_table"] + more_tol + 3 * O.F32 * total.abs()).all())
    assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in (q, k, v))


@pytest.mark.parametrize("heads,kv_heads,dim,spec", [(16, 1, 128, (48, 255, True)), (16, 1, 64, (48, 255, True)), (1, 1, 64, (48, 4000, True)),
                                                     (2, 2, 128, (48, 8191, False)), (9, 3, 64, (40, 300, False)), (14, 2, 96, (6, 5, True))])
def test_largest_bias_tables(dev, heads, kv_heads, dim, spec):
    """Tables that take all the room there is for them, and groups that do not
    divide a warp."""
    p = problem(dev, [330, 1, 140], [330, 400, 61], heads=heads, kv_heads=kv_heads, dim=dim, spec=spec, table_dtype=torch.float32)
    check(call(p, False, True), p, False)
