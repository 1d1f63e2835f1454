"""The packed attention and the relative position bias without a GPU: bucket
borders, refusals, and the 64-bit oracle against differences."""
import ctypes
import math

import pytest
import torch

from oracle import packed as O


@pytest.mark.parametrize("spec", [(32, 128, True), (32, 128, False), (16, 64, True), (48, 300, False), (64, 800, True),
                                  (4, 2, True), (2, 2, False), (32, 17, False), (256, 2048, True)])
def test_borders_match_the_formula(spec):
    import mergenet_b200 as mn
    b = mn.RelativeBuckets(*spec)
    side = spec[0] // 2 if spec[2] else spec[0]
    assert len(b.borders) == side - 1 and list(b.borders) == sorted(b.borders)
    for n in range(0, spec[1] + 40):
        want = O.bucket(-n, *spec)
        assert sum(x <= n for x in b.borders) == want
        exact = side // 2
        if n >= exact and side > exact:  # the usual floating formula, away from the borders
            f = math.log(n / exact) / math.log(spec[1] / exact) * (side - exact)
            if abs(f - round(f)) > 1e-9:
                assert want == min(side - 1, exact + int(f))


def test_exact_borders_are_not_rounded_away():
    """Two-sided, 32 buckets to 128: 8 * 16^(k/8) is whole for even k, and the
    bucket begins there, not one later."""
    import mergenet_b200 as mn
    b = mn.RelativeBuckets(32, 128, True)
    assert b.borders[7] == 8 and {16, 32, 64} <= set(b.borders)


@pytest.mark.parametrize("bad", [dict(num_buckets=1, two_sided=False), dict(num_buckets=2), dict(num_buckets=33),
                                 dict(max_distance=8), dict(max_distance=1 << 21), dict(num_buckets=True),
                                 dict(num_buckets=32.0), dict(num_buckets=512)])
def test_bucket_refusals(bad):
    import mergenet_b200 as mn
    with pytest.raises(ValueError):
        mn.RelativeBuckets(**bad)


def _call(**kw):
    import mergenet_b200 as mn
    t = dict(q=torch.zeros(6, 4, 64, dtype=torch.float16), k=torch.zeros(6, 2, 64, dtype=torch.float16),
             v=torch.zeros(6, 2, 64, dtype=torch.float16), cu_seqlens_q=torch.tensor([0, 2, 6], dtype=torch.int32))
    t.update(kw)
    return mn.packed_attention(**t)


def _half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


@pytest.mark.parametrize("kw,match", [
    (dict(q=_half(6, 256)), "rows, heads, head_dim"),
    (dict(v=_half(6, 2, 32)), "shape mismatch"),
    (dict(q=_half(6, 4, 32)), "shape mismatch"),
    (dict(q=_half(6, 4, 64).bfloat16()), "share a dtype"),
    (dict(q=_half(6, 4, 64).float(), k=_half(6, 2, 64).float(), v=_half(6, 2, 64).float()), "float16 or bfloat16"),
    (dict(q=_half(6, 3, 64)), "multiple of the 2 key heads"),
    (dict(q=_half(6, 4, 136), k=_half(6, 2, 136), v=_half(6, 2, 136)), "head_dim 136"),
    (dict(q=_half(6, 4, 20), k=_half(6, 2, 20), v=_half(6, 2, 20)), "head_dim 20"),
    (dict(q=_half(6, 258, 8), k=_half(6, 2, 8), v=_half(6, 2, 8)), "at most 128"),
    (dict(k=_half(7, 2, 64), v=_half(7, 2, 64)), "queries' rows"),
    (dict(cu_seqlens_q=torch.tensor([0, 2, 6])), "int32"),
    (dict(cu_seqlens_q=torch.zeros(1, dtype=torch.int32)), "at least two"),
    (dict(cu_seqlens_k=torch.tensor([0, 6], dtype=torch.int32)), "3 entries"),
    (dict(lengths_k=torch.tensor([2], dtype=torch.int32)), "2 entries"),
    (dict(scale=0.0), "positive"),
    (dict(scale=float("nan")), "positive"),
    (dict(bias_table=_half(32, 4)), "go together"),
])
def test_argument_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _call(**kw)


def test_bias_refusals():
    import mergenet_b200 as mn
    b = mn.RelativeBuckets(32, 128)
    with pytest.raises(ValueError, match="bias table"):
        _call(bias_table=_half(32, 3), buckets=b)
    with pytest.raises(ValueError, match="bias table"):
        mn.relative_position_bias(_half(16, 3), 2, 2, b)
    with pytest.raises(TypeError, match="RelativeBuckets"):
        mn.relative_position_bias(_half(32, 3), 2, 2, 32)
    with pytest.raises(TypeError, match="dtype"):
        mn.relative_position_bias(torch.zeros(32, 3, dtype=torch.float64), 2, 2, b)
    with pytest.raises(ValueError, match="does not fit"):
        _call(bias_table=_half(32, 4), buckets=mn.RelativeBuckets(32, 8192))
    with pytest.raises(ValueError, match="does not fit"):
        _call(bias_table=_half(96, 4), buckets=mn.RelativeBuckets(96, 128))
    with pytest.raises(ValueError, match="does not fit"):
        _call(q=_half(6, 34, 64), k=_half(6, 2, 64), v=_half(6, 2, 64), bias_table=_half(32, 34), buckets=b)
    with pytest.raises(ValueError, match="2\\^30"):
        mn.relative_position_bias(_half(32, 3), 2, 2, b, query_start=1 << 30)
    with pytest.raises(ValueError, match="negative"):
        mn.relative_position_bias(_half(32, 3), -1, 2, b)


def test_host_tensors_are_refused():
    import mergenet_b200 as mn
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mn.relative_position_bias(_half(32, 3), 2, 2, mn.RelativeBuckets(32, 128))


def test_c_entry_points_refuse_bad_arguments():
    """The C entry points return a status before anything is launched."""
    from mergenet_b200 import _lib as L
    lib = L.lib()
    a = L.PackedArgs()
    assert lib.mn_packed_attention(ctypes.byref(a), None, 0, None, None) == L.MN_ERR_ARG
    assert lib.mn_packed_attention(None, None, 0, None, None) == L.MN_ERR_ARG
    buf = (ctypes.c_int32 * 4)()
    at = ctypes.addressof(buf)
    for n in ("q", "k", "v", "cu_q", "cu_k", "out"):
        setattr(a, n, at)
    a.nseq, a.tq, a.tk, a.heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 1, 1, 1, 1, 1, 64, L.MN_F32, 1.0
    assert lib.mn_packed_attention(ctypes.byref(a), None, 0, None, None) == L.MN_ERR_UNSUPPORTED
    a.dtype, a.head_dim = L.MN_F16, 129
    assert lib.mn_packed_attention(ctypes.byref(a), None, 0, None, None) == L.MN_ERR_UNSUPPORTED
    a.head_dim, a.bias_table, a.buckets, a.num_borders, a.borders = 64, at, 4, 3, at  # borders must be >= 1
    assert lib.mn_packed_attention(ctypes.byref(a), None, 0, None, None) == L.MN_ERR_ARG
    assert lib.mn_packed_attention_backward(ctypes.byref(a), None, 0, None, None) == L.MN_ERR_ARG
    assert lib.mn_relative_bias(0, 1, 1, 0, 2, 0, 1, at, 0, at, at, None) == L.MN_ERR_ARG
    assert lib.mn_relative_bias(1, 1, 1, 0, 2, 0, 0, at, 0, at, at, None) == L.MN_ERR_ARG


@pytest.mark.parametrize("causal,biased", [(False, False), (True, True), (False, True)])
def test_oracle_gradients_match_differences(causal, biased):
    """Each gradient of the 64-bit oracle against central differences of its
    own forward."""
    gen = torch.Generator().manual_seed(5)
    nq, nk, spec = [3, 0, 4, 2], [2, 3, 5, 0], (8, 6, True)
    q = torch.randn(9, 4, 8, generator=gen, dtype=torch.float64)
    k = torch.randn(10, 2, 8, generator=gen, dtype=torch.float64)
    v = torch.randn(10, 2, 8, generator=gen, dtype=torch.float64)
    w = torch.randn(9, 4, 8, generator=gen, dtype=torch.float64)
    table = torch.randn(8, 4, generator=gen, dtype=torch.float64) if biased else None
    O.HALF_STEP[torch.float64], O.TINY[torch.float64] = 0.0, 0.0
    try:
        kw = dict(nq=nq, nk=nk, causal=causal, spec=spec)
        val, _ = O.packed_attention(q, k, v, table=table, dout=w, **kw)
        for name, x in (("grad_q", q), ("grad_k", k), ("grad_v", v)) + ((("grad_table", table),) if biased else ()):
            for _ in range(4):
                step = torch.randn(x.shape, generator=gen, dtype=torch.float64)
                sides = []
                for sign in (1e-4, -1e-4):
                    at = {"grad_q": q, "grad_k": k, "grad_v": v, "grad_table": table}
                    at[name] = x + sign * step
                    o, _ = O.packed_attention(at["grad_q"], at["grad_k"], at["grad_v"], table=at["grad_table"], **kw)
                    sides.append(float((o["out"] * w).sum()))
                want = (sides[0] - sides[1]) / 2e-4
                # the difference is off by h^2 / 6 of a third derivative of order 10^2, and by 2^-53 / h
                assert abs(float((val[name] * step).sum()) - want) < 1e-5
    finally:
        del O.HALF_STEP[torch.float64], O.TINY[torch.float64]
