"""Uses of the packed attention and the relative position bias at the edge of
what they accept, without a GPU."""
import ctypes
import types

import pytest
import torch


def _check_status(monkeypatch, word):
    import mergenet_b200 as mn
    from mergenet_b200.model import MergeNetSmall
    monkeypatch.setattr(mn.attention, "attention_status", lambda device=None, reset=False: word)
    MergeNetSmall.check_status(types.SimpleNamespace(), torch.zeros(1, dtype=torch.int32))


def test_bad_offsets_of_another_call_are_not_the_models_error(monkeypatch):
    from mergenet_b200 import _lib as L
    _check_status(monkeypatch, 0)
    _check_status(monkeypatch, L.MN_STATUS_BAD_LENGTHS)


@pytest.mark.parametrize("more", [0, 512])
def test_a_models_status_names_the_timeout(monkeypatch, more):
    from mergenet_b200 import _lib as L
    with pytest.raises(RuntimeError, match="0x100 .*gave up"):
        _check_status(monkeypatch, L.MN_STATUS_TC_TIMEOUT | more)
    with pytest.raises(RuntimeError, match="unknown"):
        _check_status(monkeypatch, 1 << 20 | more)


def _c_args(backward=False, **kw):
    """Arguments of a call that divides its keys, on addresses that are never read."""
    from mergenet_b200 import _lib as L
    a = L.PackedArgs()
    for i, n in enumerate(("q", "k", "v", "cu_q", "cu_k", "out", "lse") + (("dout", "dq", "dk", "dv") if backward else ())):
        setattr(a, n, 1 << 20 | i << 12)
    a.nseq, a.tq, a.tk, a.heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 1, 1, 20000, 4, 2, 128, L.MN_F16, 1.0
    a.q_st = a.do_st = 512
    a.k_st = a.v_st = 256
    a.q_sh = a.k_sh = a.v_sh = a.do_sh = 128
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_c_entry_refuses_unaligned_tensors(name):
    """Rows are read and written 16 bytes at a time: nothing is launched on an
    address that is not a multiple (the size of the workspace is 0 for calls
    that are refused)."""
    from mergenet_b200 import _lib as L
    size = L.lib().mn_packed_attention_workspace_bytes
    assert size(ctypes.byref(_c_args())) > 0
    for off in (2, 4, 8):
        a = _c_args(**{name: (1 << 20) + off})
        assert size(ctypes.byref(a)) == 0
        assert L.lib().mn_packed_attention(ctypes.byref(a), 1 << 21, 1 << 40, None, None) == L.MN_ERR_UNSUPPORTED


@pytest.mark.parametrize("name", ["q", "k", "v", "out", "dout", "dq", "dk", "dv"])
def test_c_entry_refuses_unaligned_gradients(name):
    from mergenet_b200 import _lib as L
    size = L.lib().mn_packed_attention_backward_workspace_bytes
    assert size(ctypes.byref(_c_args(True))) > 0
    a = _c_args(True, **{name: (1 << 20) + 8})
    assert size(ctypes.byref(a)) == 0
    assert L.lib().mn_packed_attention_backward(ctypes.byref(a), 1 << 21, 1 << 40, None, None) == L.MN_ERR_UNSUPPORTED


def test_c_entry_refuses_an_unaligned_workspace():
    from mergenet_b200 import _lib as L
    lib = L.lib()
    assert lib.mn_packed_attention(ctypes.byref(_c_args()), (1 << 21) + 8, 1 << 40, None, None) == L.MN_ERR_WORKSPACE
    assert lib.mn_packed_attention_backward(ctypes.byref(_c_args(True)), (1 << 21) + 8, 1 << 40, None, None) == L.MN_ERR_WORKSPACE
    at = ctypes.addressof((ctypes.c_int32 * 1)(1))
    assert lib.mn_relative_bias_backward(1, 4, 4, 0, 2, 0, 1, at, 0, 1 << 20, 1 << 20, (1 << 21) + 2, 1 << 40, None) == L.MN_ERR_WORKSPACE


@pytest.mark.parametrize("sizes,match", [
    (dict(tq=1 << 20, tk=1 << 20, heads=4096, kv_heads=4096), "2\\^31 query rows"),
    (dict(tq=1 << 29, tk=1 << 29, heads=4, kv_heads=4), "2\\^31 query rows"),
    (dict(tq=1, tk=1, heads=65535, kv_heads=65535, nseq=1 << 15), "2\\^31 tiles"),
    (dict(tq=1, tk=1 << 29, heads=1024, kv_heads=1024), "2\\^31 tiles"),
    (dict(tq=1, tk=1 << 30, heads=1, kv_heads=1), "2\\^30 rows"),
])
def test_sizes_past_a_launch_are_refused_beforehand(sizes, match):
    """By name in Python, and before anything is launched in C."""
    import mergenet_b200 as mn
    from mergenet_b200 import _lib as L
    nseq = sizes.get("nseq", 1)
    meta = [torch.empty(sizes[r], sizes[h], 8, dtype=torch.float16, device="meta")
            for r, h in (("tq", "heads"), ("tk", "kv_heads"), ("tk", "kv_heads"))]
    cu = torch.empty(nseq + 1, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match=match):
        mn.packed_attention(*meta, cu, cu)
    h, hk = sizes["heads"], sizes["kv_heads"]
    a = _c_args(True, **sizes, head_dim=8, q_st=8 * h, do_st=8 * h, k_st=8 * hk, v_st=8 * hk, q_sh=8, k_sh=8, v_sh=8, do_sh=8)
    assert L.lib().mn_packed_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
    assert L.lib().mn_packed_attention(ctypes.byref(a), 1 << 21, 1 << 40, None, None) == L.MN_ERR_UNSUPPORTED


@pytest.mark.parametrize("sizes", [dict(tq=1 << 19, tk=1 << 19, heads=4095, kv_heads=4095), dict(tq=1, tk=1 << 28, heads=8, kv_heads=8),
                                   dict(tq=1, tk=1, heads=65535, kv_heads=65535, nseq=32000)])
def test_the_largest_sizes_are_not(sizes):
    from mergenet_b200 import _lib as L
    import mergenet_b200 as mn
    h, hk = sizes["heads"], sizes["kv_heads"]
    a = _c_args(True, **sizes, head_dim=8, q_st=8 * h, do_st=8 * h, k_st=8 * hk, v_st=8 * hk, q_sh=8, k_sh=8, v_sh=8, do_sh=8)
    assert L.lib().mn_packed_attention_backward_workspace_bytes(ctypes.byref(a)) > 0
    meta = [torch.empty(sizes[r], sizes[n], 8, dtype=torch.float16, device="meta")
            for r, n in (("tq", "heads"), ("tk", "kv_heads"), ("tk", "kv_heads"))]
    cu = torch.empty(sizes.get("nseq", 1) + 1, dtype=torch.int32, device="meta")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):  # all that is wrong with it
        mn.packed_attention(*meta, cu, cu)


@pytest.mark.parametrize("kw", [dict(k_sh=1 << 32, v_sh=1 << 31), dict(q_sh=1 << 35, do_sh=(1 << 31) + 8), dict(q_st=1 << 38),
                                dict(heads=1, kv_heads=1, q_sh=1 << 45, k_sh=1 << 45), dict(tq=1, q_st=1 << 45)])
def test_c_entry_takes_any_stride_of_a_tensor(kw):
    """Strides past 2^31 (a cache laid out head by head), and any stride of a
    dimension of one."""
    from mergenet_b200 import _lib as L
    assert L.lib().mn_packed_attention_backward_workspace_bytes(ctypes.byref(_c_args(True, **dict(dict(tq=2), **kw)))) > 0


@pytest.mark.parametrize("kw", [dict(k_sh=1 << 39), dict(q_sh=1 << 38), dict(k_sh=-128), dict(q_st=0), dict(v_sh=4), dict(k_st=1 << 39)])
def test_c_entry_refuses_strides_that_no_tile_map_has(kw):
    from mergenet_b200 import _lib as L
    assert L.lib().mn_packed_attention_backward_workspace_bytes(ctypes.byref(_c_args(True, **dict(dict(tq=2), **kw)))) == 0


@pytest.mark.parametrize("scale", [1e39, 3.5e38, 1e-46, 5e-324, -1.0, float("inf")])
def test_scales_that_fp32_does_not_have_are_refused(scale):
    import mergenet_b200 as mn
    x = torch.zeros(6, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="scale must be positive"):
        mn.packed_attention(x, x, x, torch.tensor([0, 6], dtype=torch.int32), scale=scale)


@pytest.mark.parametrize("spec", [(32, 128, True), (48, 700, False)])
def test_buckets_are_saved_and_copied(spec):
    """With a module that holds them, or to another process."""
    import copy
    import io
    import pickle
    import mergenet_b200 as mn
    b = mn.RelativeBuckets(*spec)
    module = torch.nn.Module()
    module.buckets = b
    file = io.BytesIO()
    torch.save(module, file)
    file.seek(0)
    for c in (pickle.loads(pickle.dumps(b)), copy.deepcopy(b), copy.copy(b), torch.load(file, weights_only=False).buckets):
        assert repr(c) == repr(b) and c.borders == b.borders and list(c._c_borders) == list(b.borders)


# ------------------------------------------------- what the GPU tests' bounds catch
BOUND_SHAPES = [([200, 520], 16, 1, 128, (32, 128, True)), ([200, 520], 6, 6, 64, (32, 128, True)), ([300, 1, 129], 4, 2, 64, (32, 128, False))]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,heads,kv_heads,dim,spec", BOUND_SHAPES)
def test_bounds_reject_results_that_are_off(nq, heads, kv_heads, dim, spec, dtype, causal):
    """The bounds that add roundings by their squares: a result of another
    factor, a head or a sum by bucket left out, a table that lost its outermost
    buckets and a key too few are rejected."""
    from oracle import packed as O
    gen = torch.Generator().manual_seed(0)
    t = {n: torch.randn(sum(nq), h, dim, generator=gen).to(dtype) for n, h in
         (("q", heads), ("k", kv_heads), ("v", kv_heads), ("dout", heads))}
    table = torch.randn(spec[0], heads, generator=gen)

    def run(f, nk=nq, dout=t["dout"], table=table):
        return f(t["q"], t["k"], t["v"], nq, nk, nq, causal=causal, table=table, spec=None if table is None else spec, dout=dout)

    val, tol = run(O.packed_attention_spread)
    first, _ = run(O.packed_attention)
    for n in val:
        assert torch.allclose(val[n], first[n], rtol=1e-12, atol=1e-12), n
    passes = lambda n, x: bool(((x - val[n]).abs() <= tol[n]).all())  # noqa: E731
    for n in val:
        assert passes(n, val[n])
        assert not passes(n, 0.95 * val[n]) and not passes(n, 1.05 * val[n]), n
    far = [spec[0] // 2 - 1] + ([] if causal else [spec[0] - 1]) if spec[2] else [spec[0] - 1]
    for bucket in far:
        x = val["grad_table"].clone()
        x[bucket] = 0
        assert not passes("grad_table", x), bucket
    less = t["dout"].clone()
    less[:, heads - 1] = 0  # the last head's share of the gradients
    part, _ = run(O.packed_attention, dout=less)
    for n in ("grad_q", "grad_k", "grad_v", "grad_table"):
        assert not passes(n, part[n]), n
    plain, plain_tol = run(O.packed_attention_spread, table=None)
    fewer, _ = run(O.packed_attention, nk=[max(0, x - 1) for x in nq], table=None)
    if not causal:  # under the causal mask the positions move along
        for n in plain:
            assert bool(((fewer[n] - plain[n]).abs() > plain_tol[n]).any()), n
