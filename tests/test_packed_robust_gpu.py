"""The packed attention beside other calls and at the edge of what it accepts,
on the GPU."""
import pytest
import torch

from oracle import packed as O
from test_packed_gpu import SPEC, call, check, offsets, problem

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("bad", ["past_the_end", "descending", "first", "length"])
def test_a_call_with_bad_offsets_leaves_later_calls_alone(dev, bad):
    """Bad offsets are recorded in a word that other attention calls share and
    that stays set; what those calls return is what they return without it."""
    import mergenet_b200 as mn
    from mergenet_b200 import _lib as L
    from mergenet_b200 import attention as local
    train = problem(dev, [2500, 1, 600], heads=16, kv_heads=4, dim=128, dtype=torch.bfloat16)
    images = problem(dev, [785, 393, 500], heads=6, kv_heads=6, dtype=torch.float16, spec=SPEC)
    cache = problem(dev, [1, 1], [30000, 700], heads=8, kv_heads=2, dim=128)
    gen = torch.Generator(device=dev).manual_seed(0)
    q, k, v = (torch.randn(4, 785, 6, 64, generator=gen, device=dev).half() for _ in range(3))
    qkv = torch.randn(4, 785, 3 * 384, generator=gen, device=dev).half()
    latent = torch.randn(4, 100, 6, 64, generator=gen, device=dev).half()

    def valid():
        got = [call(train, True, True), call(images, False, True), call(cache, True, False)]
        got.append({"local": local.unbiased_local_attention(q, k, v, 16),
                    "wide": local.unbiased_local_attention(q, k, v, 64),
                    "packed": local.local_attention_packed(qkv, 6, 16)})
        got.append({"latent": local.local_attention_packed(qkv, 6, -1), "cross": local.cross_attention(latent, k, v)})
        return got

    want = valid()
    p = problem(dev, [30, 40])
    cu, lens = {"past_the_end": ([0, 30, 900], None), "descending": ([0, 50, 20], None), "first": ([3, 30, 70], None),
                "length": ([0, 30, 70], [31, -1])}[bad]
    leaf = p["q"].detach().requires_grad_(True)
    mn.packed_attention(leaf, p["k"], p["v"], torch.tensor(cu, dtype=torch.int32, device=dev),
                        lengths_k=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)).sum().backward()
    assert mn.attention.attention_status(dev) == L.MN_STATUS_BAD_LENGTHS
    for _ in range(3):
        for a, b in zip(valid(), want):
            for name in b:
                assert torch.equal(a[name], b[name]), name
    assert mn.attention.attention_status(dev, reset=True) == L.MN_STATUS_BAD_LENGTHS


# ------------------------------------------- gradients in the range of fp16
def _scaled(p, **factors):
    for name, f in factors.items():
        p[name] = (p[name].float() * f).to(p[name].dtype)
    return p


@pytest.mark.parametrize("spec", [None, SPEC])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 2, 128), (8, 1, 64)])
def test_score_gradients_past_the_range_of_fp16(dev, heads, kv_heads, dim, spec):
    """Upstream gradients of a large loss scale: dq, dk and dv fit fp16, while
    p (dp - delta) reaches 2 x 10^5 and more."""
    p = problem(dev, [300, 1, 150], heads=heads, kv_heads=kv_heads, dim=dim, dtype=torch.float16, spec=spec, table_dtype=torch.float32)
    _scaled(p, q=1 / 16, k=1 / 16, v=16, dout=4096)
    check(call(p, True, True), p, True)


def _relative(x, want):
    return float((x.double() - want).norm() / want.norm())


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 2, 128), (2, 1, 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("name,factors", [("grad_q", dict(k=64, q=1 / 64)), ("grad_k", dict(q=64, k=1 / 64))])
def test_small_upstream_gradients_in_fp16(dev, name, factors, causal, heads, kv_heads, dim):
    """Upstream gradients of 2^-12 over 1,500 keys: p (dp - delta) is about
    2^-20, where fp16 has steps of 2^-24; the gradients that it gives (about
    2^-12, the keys or queries being large) are good to fp16's own step.

    A term is rounded once (2^-11 at most, 2^-11 / sqrt(3) in the mean square)
    and so is the result; both together come to 2^-11 of the norm.  The bound
    is four times that.  Terms rounded in steps of 2^-24 would be off by
    2^-26 or more each, 2^-6 of the norm."""
    p = _scaled(problem(dev, [1500], heads=heads, kv_heads=kv_heads, dim=dim, dtype=torch.float16), dout=2.0 ** -12, **factors)
    got = call(p, causal, True)
    val, _ = O.packed_attention(p["q"], p["k"], p["v"], p["nq"], p["nk"], causal=causal, dout=p["dout"])
    assert _relative(got[name], val[name]) < 2.0 ** -9
    assert _relative(got["grad_v"], val["grad_v"]) < 2.0 ** -9 + 2.0 ** -25 * val["grad_v"].numel() ** 0.5 / float(val["grad_v"].norm())


def test_values_of_little_weight_in_fp16(dev):
    """A key whose weight is 2^-21 for every query, under upstream gradients of
    2^10: its dv is within the normal range of fp16.  Each of the weights is
    rounded by 2^-11 relative, is off by 2 E through the scores (66 products:
    72 x 2^-24 x 2 x 7.5 x 2) and 2^-16 through the exponential, and the result
    is rounded once more."""
    n = 64
    p = problem(dev, [n], [2], heads=2, kv_heads=2, dtype=torch.float16)
    p["q"] = (1 + 0.02 * p["q"].float()).half()
    p["k"] = torch.full_like(p["k"], 0.9375)
    p["k"][1] *= -1
    _scaled(p, dout=1024)
    got = call(p, False, True)["grad_v"]
    val, _ = O.packed_attention(p["q"], p["k"], p["v"], [n], [2], dout=p["dout"])
    weight = torch.softmax(torch.einsum("ihd,jhd->hij", p["q"].double(), p["k"].double()) / 8, -1)
    assert float(weight[..., 1].max()) < 2.0 ** -18 and float(weight[..., 1].min()) > 2.0 ** -25
    mag = torch.einsum("hij,ihd->jhd", weight, p["dout"].double().abs())
    assert ((got.double() - val["grad_v"]).abs() <= (2.0 ** -11 + 72 * 2.0 ** -24 * 30 + 2.0 ** -16) * mag
            + 2.0 ** -11 * val["grad_v"].abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_the_range_of_other_rows_reaches_nothing(dev, dim):
    """Large finite values in another sequence, in unused cache rows and behind
    the last sequence change no bit of a sequence's gradients."""
    nq, nk, slots = [70, 50, 131], [70, 60, 131], [100, 128, 256]
    p = problem(dev, nq, nk, slots, dim=dim, dtype=torch.float16, spec=SPEC, extra=40)
    lens = torch.tensor(nk, dtype=torch.int32, device=dev)
    clean = call(p, False, True, lengths=lens)
    for n in ("q", "dout"):
        p[n][70:120] *= 2.0 ** 12
        p[n][251:] = 60000.0
    p["k"][100:228] = 1.5
    for n in ("k", "v"):
        p[n][70:100] = 60000.0
        p[n][100:228] = p[n][100:228].abs() + 512
        p[n][228 + 131:] = -60000.0
    got = call(p, False, True, lengths=lens)
    rows = torch.cat([torch.arange(70), torch.arange(120, 251)]).to(dev)
    keys = torch.cat([torch.arange(70), torch.arange(228, 359)]).to(dev)
    for n in ("out", "grad_q"):
        assert torch.equal(got[n][rows], clean[n][rows]), n
    for n in ("grad_k", "grad_v"):
        assert torch.equal(got[n][keys], clean[n][keys]), n


def test_gradients_of_zero_and_of_one_value_in_fp16(dev):
    """Ranges without a value to go by: no upstream gradient, no values, the
    smallest and the largest ones that fp16 has."""
    p = problem(dev, [140, 30], heads=4, kv_heads=2, dtype=torch.float16)
    for n in ("dout", "v"):
        got = call(dict(p, **{n: torch.zeros_like(p[n])}), True, True)
        assert not got["grad_q"].any() and not got["grad_k"].any()
        assert (n == "v") == bool(got["grad_v"].any())
    for dout, v in ((2.0 ** -24, 2.0 ** -24), (65504.0, 2.0 ** -24), (2.0 ** -24, 65504.0)):
        one = dict(p, dout=torch.sign(p["dout"]) * dout, v=torch.sign(p["v"]) * v)
        got = call(one, False, True)
        val, tol = O.packed_attention(one["q"], one["k"], one["v"], one["nq"], one["nk"], dout=one["dout"])
        for n, x in got.items():  # a key that many queries weigh highest may have a dv past fp16's range
            fits = val[n].abs() + tol[n] < 65504
            assert ((x.double() - val[n]).abs() <= tol[n])[fits].all(), n
            assert (torch.isinf(x) | ((x.double() - val[n]).abs() <= tol[n]))[~fits].all(), n
            assert float(fits.double().mean()) > 0.99


# ------------------------------------------------------ forward-mode tangents
@pytest.mark.parametrize("which", ["q", "k", "v", "table"])
def test_forward_mode_tangents_are_refused(dev, which):
    """Not dropped: the same error with and without a gradient asked for."""
    import mergenet_b200 as mn
    from torch.autograd import forward_ad
    p = problem(dev, [20], spec=SPEC)
    buckets, cu = mn.RelativeBuckets(*SPEC), offsets([20], dev)

    def run(x):
        out = mn.packed_attention(x["q"], x["k"], x["v"], cu, bias_table=x["table"], buckets=buckets)
        return out, mn.relative_position_bias(x["table"], 4, 4, buckets)

    want = run(p)
    for grad in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(p[which].detach().requires_grad_(grad), torch.ones_like(p[which]))
            with pytest.raises(NotImplementedError, match="jvp"):
                mn.packed_attention(*(dual if n == which else p[n] for n in ("q", "k", "v")), cu,
                                    bias_table=dual if which == "table" else p["table"], buckets=buckets)
            if which == "table":
                with pytest.raises(NotImplementedError, match="jvp"):
                    mn.relative_position_bias(dual, 4, 4, buckets)
    with forward_ad.dual_level():  # no tangent on these
        for a, b in zip(run(p), want):
            assert torch.equal(a, b) and not a.requires_grad
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(p["q"], torch.ones_like(p["q"]))
        with pytest.raises(NotImplementedError, match="jvp"):
            mn.packed_attention(dual, p["k"], p["v"], cu)


def test_function_transforms_are_refused(dev):
    """torch.func's wrappers have no memory that a kernel could read."""
    import mergenet_b200 as mn
    p = problem(dev, [20])
    cu = offsets([20], dev)
    f = lambda q: mn.packed_attention(q, p["k"], p["v"], cu)  # noqa: E731
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (p["q"],), (torch.ones_like(p["q"]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(p["q"][None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda q: f(q).float().sum())(p["q"])


# ----------------------------------------------------------------- layouts
def test_head_strides_past_32_bits(dev):
    """Keys, values, queries and their gradient laid out head by head, the
    heads more than 2^31 values apart; only their rows are ever written."""
    import mergenet_b200 as mn
    p = problem(dev, [70, 3], [300, 77], heads=2, kv_heads=2, dim=64)
    want = call(p, True, True)
    apart = (1 << 31) + 64
    memory = torch.empty(apart + (1 << 18), device=dev, dtype=torch.bfloat16)
    at, wide = 0, {}
    for n in ("q", "k", "v", "dout"):
        rows = p[n].shape[0]
        wide[n] = memory.as_strided((rows, 2, 64), (64, apart, 1), at)
        wide[n].copy_(p[n])
        at += rows * 64
    assert wide["k"].stride(1) > 1 << 31
    leaves = [wide[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
    out = mn.packed_attention(*leaves, offsets(p["nq"], dev), offsets(p["nk"], dev), causal=True)
    got = [out.detach(), *torch.autograd.grad(out, leaves, wide["dout"])]
    for x, n in zip(got, want):
        assert torch.equal(x, want[n]), n


def test_any_stride_of_a_dimension_of_one(dev):
    import mergenet_b200 as mn
    p = problem(dev, [70], heads=1, kv_heads=1)
    want = call(p, True, True)
    leaves = [p[n].as_strided(p[n].shape, (64, 1 << 45, 1)).requires_grad_(True) for n in ("q", "k", "v")]
    out = mn.packed_attention(*leaves, offsets([70], dev), causal=True)
    got = [out.detach(), *torch.autograd.grad(out, leaves, p["dout"])]
    for x, n in zip(got, want):
        assert torch.equal(x, want[n]), n
