"""The forms of the packed attention's kernels that its sizes choose (keys
divided or not, tiles by work or in order, one or two tiles a CTA, with and
without a bias, both types), within bounds that add roundings by their squares
(oracle.packed.packed_attention_spread)."""
import random

import pytest
import torch

from oracle import packed as O
from test_packed_gpu import LENGTHS, SPEC, call, offsets, problem, randn

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


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


def check(got, p, causal, scale=None):
    val, tol = O.packed_attention_spread(p["q"], p["k"], p["v"], p["nq"], p["nk"], p["slots"], causal=causal, scale=scale,
                                         table=p["table"], spec=p["spec"], dout=p["dout"] if "grad_q" in got else None)
    for name, x in got.items():
        assert torch.isfinite(x.float()).all(), name
        if x.numel():
            off = (x.double() - val[name]).abs()
            worst = (off - tol[name]).argmax()
            assert bool((off <= tol[name]).all()), \
                f"{name}: {float(off.flatten()[worst]):.3e} off, bound {float(tol[name].flatten()[worst]):.3e}"


def divided(p, lengths=None):
    """The forward call divides its keys (only then has it a workspace)."""
    from mergenet_b200 import _lib as L
    from mergenet_b200 import RelativeBuckets, packed
    dev = p["q"].device
    cu_q, cu_k = offsets(p["nq"], dev), offsets(p["slots"], dev)
    out = torch.empty_like(p["q"])
    args = packed._args(p["q"], p["k"], p["v"], cu_q, cu_k, lengths, True, 1.0, p["table"],
                        RelativeBuckets(*p["spec"]) if p["spec"] else None, out, None)
    return L.lib().mn_packed_attention_workspace_bytes(args) > 0


@BOTH
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_lengths(dev, lengths, dim, causal, dtype):
    nq, nk = LENGTHS[lengths]
    p = problem(dev, nq, nk, dim=dim, dtype=dtype)
    check(call(p, causal, True), p, causal)


@BOTH
@pytest.mark.parametrize("heads,kv_heads,dim,spec,table_dtype", [
    (32, 2, 64, SPEC, torch.float32), (16, 1, 128, SPEC, torch.float32), (12, 4, 80, SPEC, torch.float32), (6, 6, 64, SPEC, torch.float16),
    (5, 1, 128, (32, 128, False), torch.float32), (14, 2, 64, (16, 40, True), torch.bfloat16), (16, 1, 128, (48, 255, True), torch.float32),
    (1, 1, 64, (48, 4000, True), torch.float32), (2, 2, 128, (48, 8191, False), torch.float32)])
@pytest.mark.parametrize("causal", [False, True])
def test_bias(dev, heads, kv_heads, dim, spec, table_dtype, causal, dtype):
    p = problem(dev, [520, 1, 200], [520, 400, 61], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, spec=spec, table_dtype=table_dtype)
    check(call(p, causal, True), p, causal)


DIVIDED = {
    "one_token": ([1], [9000]),
    "tokens": ([1, 1, 1, 1], [5000, 1, 3000, 0]),
    "a_few_tokens_each": ([3, 1, 5], [4000, 2000, 4]),
    "a_short_prompt": ([40, 7], [3000, 4097]),
    "more_queries_than_keys": ([70, 1], [20, 6000]),
    "many": ([1, 2, 0, 1] * 12, [900, 1500, 40, 700] * 12),
}


@BOTH
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (6, 6, 32), (32, 1, 64), (8, 2, 128), (7, 1, 96)])
@pytest.mark.parametrize("lengths", list(DIVIDED))
def test_divided_keys(dev, lengths, heads, kv_heads, dim, dtype):
    nq, nk = DIVIDED[lengths]
    p = problem(dev, nq, nk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    assert divided(p) or dim <= 64 and lengths == "many"
    for causal in (False, True):
        check(call(p, causal, False), p, causal)
        check(call(p, causal, True), p, causal)


@BOTH
@pytest.mark.parametrize("spec", [(32, 128, True), (32, 256, False), (48, 500, False)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (6, 6, 64), (16, 1, 128), (6, 2, 80)])
@pytest.mark.parametrize("lengths", ["one_token", "a_few_tokens_each", "a_short_prompt", "more_queries_than_keys"])
def test_divided_keys_with_a_bias(dev, lengths, heads, kv_heads, dim, spec, dtype):
    nq, nk = DIVIDED[lengths]
    p = problem(dev, nq, nk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, spec=spec, table_dtype=torch.float32)
    assert divided(p)
    for causal in (False, True):
        check(call(p, causal, False), p, causal)
    check(call(p, True, True), p, True)


@BOTH
@pytest.mark.parametrize("spec", [None, (32, 128, False)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (32, 8, 128), (4, 4, 128)])
def test_divided_keys_of_a_cache_in_slots(dev, heads, kv_heads, dim, spec, dtype):
    """Lengths in use, from none to the whole slot; what else lies in the slots
    reaches nothing."""
    nk, slots = [4096, 0, 1, 129, 3000], [4096] * 5
    p = problem(dev, [1] * 5, nk, slots, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, spec=spec, table_dtype=torch.float32, extra=3)
    lens = torch.tensor(nk, dtype=torch.int32, device=dev)
    assert divided(p, lens)
    got = call(p, True, False, lengths=lens)
    check(got, p, True)
    used = (torch.arange(4096, device=dev) < lens[:, None]).flatten()
    for n in ("k", "v"):
        p[n][:-3][~used] = float("nan")
        p[n][-3:] = float("inf")
    assert torch.equal(call(p, True, False, lengths=lens)["out"], got["out"])


def _sequences(seed, n, most):
    rng = random.Random(seed)
    return [rng.choice([0, 1, rng.randint(1, most), rng.randint(1, most // 8)]) for _ in range(n)]


@BOTH
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 64), (8, 8, 128), (24, 8, 64)])
@pytest.mark.parametrize("keys", ["same", "more", "fewer", "mixed"])
def test_key_tiles_by_work(dev, keys, heads, kv_heads, dim, dtype):
    """Sequences of different lengths whose key tiles are more than a wave, so
    that the tiles with the most queries start first."""
    nq = [1500, 700, 30, 0, 1, 2100]
    nk = {"same": nq, "more": [x + 65 for x in nq], "fewer": [max(0, x - 200) for x in nq], "mixed": [200, 1800, 3, 129, 1000, 1500]}[keys]
    assert (sum(nk) // 128 + len(nk)) * kv_heads > 148
    p = problem(dev, nq, nk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    for causal in (False, True):
        check(call(p, causal, True), p, causal)


@BOTH
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 64), (16, 4, 128)])
@pytest.mark.parametrize("n,most", [(20, 40000), (60, 4000), (255, 4000), (256, 4000)])
def test_query_tiles_by_work(dev, n, most, heads, kv_heads, dim, dtype):
    """Divided calls of more than a wave: up to 255 sequences by their keys."""
    rng = random.Random(n)
    nk = [x * 3 for x in _sequences(n, n, most)]
    nq = [1] + [rng.choice([0, 1, 1, 3]) for _ in range(n - 1)]
    p = problem(dev, nq, nk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    assert divided(p) or dim == 64 and most < 40000  # many sequences of a few thousand keys fill the card as they are
    for causal in (False, True):
        check(call(p, causal, False), p, causal)


@pytest.mark.parametrize("seed", range(40))
def test_any_call(dev, seed):
    """Calls drawn over the sizes, groups, types, lengths and masks."""
    rng = random.Random(1000 + seed)
    kv_heads, group = rng.choice([1, 2, 3, 6]), rng.choice([1, 1, 2, 3, 4, 5, 8, 13, 16, 33])
    dim = rng.choice([8, 16, 40, 64, 64, 72, 128, 128])
    dtype = rng.choice([torch.float16, torch.bfloat16])
    n = rng.choice([1, 2, 5, 40])
    nq = _sequences(rng.random(), n, rng.choice([20, 300, 900]))
    nk = rng.choice([nq, [max(0, x + rng.choice([-70, 1, 64, 300])) for x in nq], _sequences(rng.random(), n, 900)])
    slots = rng.choice([nk, [x + rng.randint(0, 100) for x in nk]])
    spec = rng.choice([None, (32, 128, True), (20, 77, False), (48, 200, True)]) if group <= 16 else None
    p = problem(dev, nq, nk, slots, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, spec=spec,
                table_dtype=rng.choice([torch.float32, dtype]), extra=rng.choice([0, 3, 200]), seed=seed)
    lens = torch.tensor(nk, dtype=torch.int32, device=dev)
    causal, scale = rng.random() < 0.5, rng.choice([None, None, 0.05, 0.4])
    check(call(p, causal, rng.random() < 0.7, scale=scale, lengths=lens), p, causal, scale)


@pytest.mark.parametrize("spec", [None, SPEC])
def test_captured_fp16_gradients(dev, spec):
    """Two captured training calls replayed in turn on inputs of very different
    range: each replay goes by its own inputs."""
    import mergenet_b200 as mn
    p = [problem(dev, [150, 0, 60], heads=4, kv_heads=2, dtype=torch.float16, spec=spec, seed=s) for s in (1, 2)]
    p[0]["dout"], p[0]["v"] = p[0]["dout"] * 4096, p[0]["v"] * 16
    p[1]["dout"] = p[1]["dout"] / 4096
    want = [call(x, True, True) for x in p]
    cu = offsets([150, 0, 60], dev)
    names = [n for n in ("q", "k", "v", "table", "dout") if p[0][n] is not None]
    graphs = []
    for i in range(2):
        still = {n: p[i][n].detach().clone() for n in names}
        leaves = [still[n].requires_grad_(True) for n in names[:-1]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mn.packed_attention(*leaves[:3], cu, causal=True, bias_table=still.get("table"),
                                      buckets=mn.RelativeBuckets(*spec) if spec else None)
            grads = torch.autograd.grad(out, leaves, still["dout"])
        graphs.append((graph, still, [out.detach(), *grads]))
    for order in ((0, 1), (1, 0), (0, 1)):
        with torch.no_grad():
            for i in order:
                for n in names:
                    graphs[i][1][n].copy_(p[order.index(i)][n])
        for i in order:
            graphs[i][0].replay()
        for i in order:
            for x, n in zip(graphs[i][2], want[0]):
                assert torch.equal(x, want[order.index(i)][n]), n


@BOTH
@pytest.mark.parametrize("tq,tk", [(0, 5), (5, 0), (0, 0)])
def test_empty_sides(dev, tq, tk, dtype):
    got = call(problem(dev, [tq], [tk], dtype=dtype), True, True)
    for n, x in got.items():
        assert not x.any(), n


def test_queries_past_32_bit_offsets(dev):
    """More than 2^31 values of queries, those at the end with keys; the others
    belong to a sequence without keys and come out as 0."""
    import mergenet_b200 as mn
    rows, h, d = (1 << 21) + 400, 8, 128
    p = problem(dev, [130, 3], [140, 300], heads=h, kv_heads=2, dim=d, dtype=torch.float16)
    q = torch.empty(rows, h, d, device=dev, dtype=torch.float16)
    dout = torch.empty(rows, h, d, device=dev, dtype=torch.float16)
    assert q.numel() > 1 << 31
    first = rows - 133
    q[:first].fill_(float("nan"))
    dout[:first].fill_(float("nan"))
    q[first:], dout[first:] = p["q"], p["dout"]
    leaves = [t.detach().requires_grad_(True) for t in (q, p["k"], p["v"])]
    out = mn.packed_attention(*leaves, torch.tensor([0, first, first + 130, rows], dtype=torch.int32, device=dev),
                              torch.tensor([0, 0, 140, 440], dtype=torch.int32, device=dev), causal=True)
    gq, gk, gv = torch.autograd.grad(out, leaves, dout)
    check({"out": out.detach()[first:], "grad_q": gq[first:], "grad_k": gk, "grad_v": gv}, p, True)
    for x in (out.detach(), gq):
        assert not x[:5000].any() and not x[first - 5000:first].any()


def test_bias_tensor_past_32_bit_offsets(dev):
    """A bias of more than 2^31 values: its last rows, and a gradient that is
    0 but for those."""
    import mergenet_b200 as mn
    h, n = 9, 15500
    b = mn.RelativeBuckets(32, 500)
    assert h * n * n > 1 << 31
    gen = torch.Generator(device=dev).manual_seed(0)
    table = randn(gen, 32, h, dtype=torch.float16).requires_grad_(True)
    bias = mn.relative_position_bias(table, n, n, b)
    last = O.relative_bias(table, 20, n, (32, 500, True))  # the queries of the last 20 positions
    assert torch.equal(bias.detach()[:, -20:], last)
    up = torch.zeros_like(bias)
    up[-1, -20:] = randn(gen, 20, n, dtype=torch.float16)
    (grad,) = torch.autograd.grad(bias, table, up)
    val, tol = O.relative_bias_grad(up[-1:, -20:], (32, 500, True), dtype=torch.float16)
    assert not grad[:, :-1].any()
    assert bool(((grad[:, -1:].double() - val).abs() <= tol).all())
