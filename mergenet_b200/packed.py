"""Attention over packed sequences of different lengths, and a learned bias
of the relative position by distance buckets.

``packed_attention`` takes the sequences of a batch laid one behind the other
(images left with different numbers of tokens after merging, documents,
prompts, or one new token each against a cache) instead of the equal lengths
of ``cross_attention`` and ``local_attention_packed``.  Heads may be grouped,
the mask may be causal, and a learned table adds a bias that depends on the
distance of query and key.  It is differentiable in q, k, v and the table.

``relative_position_bias`` writes the same bias out as a tensor, for an
attention that takes it as a mask.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .attention import _STATUS, _status

MAX_HEAD_DIM = 128
MAX_GROUP = 128       # query heads that may share a key head
MAX_BUCKETS = 48      # of a table used inside the attention
MAX_BIAS_ENTRIES = 4096  # buckets x grouped heads
MAX_BIAS_VALUES = 8192  # distances x grouped heads that a kernel keeps on chip


@functools.lru_cache(maxsize=64)
def _borders(num_buckets, max_distance, two_sided):
    side = num_buckets // 2 if two_sided else num_buckets
    exact = side // 2
    m = side - exact
    out = list(range(1, exact + 1))
    for i in range(1, m):
        # smallest n with (n / exact)^m >= (max_distance / exact)^i, by
        # bisection over whole numbers: no logarithm decides a border
        low, high = exact, max_distance
        want = max_distance ** i * exact ** m
        while low < high:
            mid = (low + high) // 2
            if mid ** m * exact ** i >= want:
                high = mid
            else:
                low = mid + 1
        out.append(low)
    return tuple(out), (ctypes.c_int32 * len(out))(*out)


class RelativeBuckets:
    """Buckets of the distance between a query and a key position.

    Distances below half of one side's buckets have a bucket each; the rest
    of the buckets divide the distances up to ``max_distance`` evenly in their
    logarithm, and the last holds everything beyond.  ``two_sided`` gives the
    keys ahead of the query the second half of the buckets; otherwise all
    keys at or ahead of the query fall into bucket 0.

    ``borders`` are the distances at which the next bucket begins.  They are
    whole numbers found without rounding: bucket ``exact + i`` begins at the
    first n with (n / exact)^m >= (max_distance / exact)^i, m the number of
    logarithmic buckets."""

    __slots__ = ("num_buckets", "max_distance", "two_sided", "borders", "_c_borders")

    def __init__(self, num_buckets=32, max_distance=128, two_sided=True):
        for name, v in (("num_buckets", num_buckets), ("max_distance", max_distance)):
            if isinstance(v, bool):
                raise ValueError(f"{name} must be an integer, got {v!r}")
            try:
                operator.index(v)
            except TypeError as exc:
                raise ValueError(f"{name} must be an integer, got {v!r}") from exc
        side = num_buckets // 2 if two_sided else num_buckets
        if side < 2 or (two_sided and num_buckets % 2):
            raise ValueError(f"num_buckets {num_buckets}: at least 2 to a side, and an even number for two sides")
        if not side // 2 < max_distance <= 1 << 20:
            raise ValueError(f"max_distance must lie in ({side // 2}, {1 << 20}], got {max_distance}")
        if side > 128:
            raise ValueError(f"num_buckets {num_buckets}: at most 128 to a side")
        self.num_buckets, self.max_distance, self.two_sided = int(num_buckets), int(max_distance), bool(two_sided)
        self.borders, self._c_borders = _borders(self.num_buckets, self.max_distance, self.two_sided)

    def __repr__(self):
        return f"RelativeBuckets({self.num_buckets}, {self.max_distance}, two_sided={self.two_sided})"


def _check_table(table, buckets, heads=None):
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError(f"buckets must be a RelativeBuckets, got {type(buckets).__name__}")
    if table.ndim != 2 or table.shape[0] != buckets.num_buckets or (heads is not None and table.shape[1] != heads):
        want = f"({buckets.num_buckets}, {'heads' if heads is None else heads})"
        raise ValueError(f"the bias table must be {want}, got {tuple(table.shape)}")
    L.dtype_code(table.dtype)


def _rows_ready(t):
    """[rows, heads, channels] with unit channel stride and rows and heads on
    16-byte boundaries (what the copies of a tile need); a broadcast
    dimension (stride 0) is laid out first."""
    st, sh, sd = t.stride()
    return (sd == 1 and st % 8 == 0 and sh % 8 == 0 and t.data_ptr() % 16 == 0 and (st > 0 or t.shape[0] == 1)
            and (sh > 0 or t.shape[1] == 1))


def _ready(t):
    return t if _rows_ready(t) else t.contiguous().clone() if t.is_contiguous() else t.contiguous()


def _err_word(dev):
    """The device's status word; none while a graph is being captured that
    would have to create it."""
    if (dev.type, dev.index) not in _STATUS and torch.cuda.is_current_stream_capturing():
        return None
    return _status(dev)


def _args(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, out, lse, dout=None, dq=None, dk=None, dv=None, dbias=None):
    """mn_packed_args in field order."""
    st = [*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *(dout.stride()[:2] if dout is not None else (0, 0))]
    pt = [0 if t is None else t.data_ptr() for t in (q, k, v, cu_q, cu_k, len_k, table)]
    po = [0 if t is None else t.data_ptr() for t in (out, lse, dout, dq, dk, dv, dbias)]
    if table is None:
        bias = (0, 0, 0, 0)
        borders = 0
    else:
        bias = (L.dtype_code(table.dtype), buckets.num_buckets, int(buckets.two_sided), len(buckets.borders))
        borders = ctypes.addressof(buckets._c_borders)
    return L.PackedArgs(*pt, borders, *po, *st, cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2],
                        L.dtype_code(q.dtype), int(causal), *bias, scale, 0)


def _workspace(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _forward(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, want_lse):
    dev = q.device
    q, k, v = _ready(q), _ready(k), _ready(v)
    out = torch.empty(q.shape, device=dev, dtype=q.dtype)
    lse = torch.empty(k.shape[1], q.shape[0], q.shape[1] // k.shape[1], device=dev, dtype=torch.float32) if want_lse else None
    table = None if table is None else table.contiguous()
    if out.numel():
        with torch.cuda.device(dev):
            lib = L.lib()
            a = _args(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, out, lse)
            nbytes = lib.mn_packed_attention_workspace_bytes(ctypes.byref(a))
            ws = _workspace(nbytes, dev)
            L.check(lib.mn_packed_attention(ctypes.byref(a), L.ptr(ws), nbytes, L.ptr(_err_word(dev)), L.stream_of(q)),
                    "mn_packed_attention")
    return out, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, len_k, causal, scale, buckets):
        out, lse = _forward(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, True)
        ctx.save_for_backward(q, k, v, table, cu_q, cu_k, len_k, out, lse)
        ctx.call = (causal, scale, buckets)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, cu_q, cu_k, len_k, out, lse = ctx.saved_tensors
        causal, scale, buckets = ctx.call
        dev = q.device
        dq = torch.empty(q.shape, device=dev, dtype=q.dtype)
        dk = torch.empty(k.shape, device=dev, dtype=k.dtype)
        dv = torch.empty(v.shape, device=dev, dtype=v.dtype)
        dbias = None if table is None else torch.empty(table.shape, device=dev, dtype=torch.float32)
        if q.numel() == 0:
            for t in (dk, dv, dbias):
                if t is not None:
                    t.zero_()
        else:
            tab = None if table is None else table.contiguous()
            qr, kr, vr, do = _ready(q), _ready(k), _ready(v), _ready(dout)
            with torch.cuda.device(dev):
                lib = L.lib()
                a = _args(qr, kr, vr, cu_q, cu_k, len_k, causal, scale, tab, buckets, out, lse, do, dq, dk, dv, dbias)
                nbytes = lib.mn_packed_attention_backward_workspace_bytes(ctypes.byref(a))
                ws = _workspace(nbytes, dev)
                L.check(lib.mn_packed_attention_backward(ctypes.byref(a), L.ptr(ws), nbytes, L.ptr(_err_word(dev)),
                                                         L.stream_of(qr)), "mn_packed_attention_backward")
        return dq, dk, dv, None if table is None else dbias.to(table.dtype), None, None, None, None, None, None


def _check_offsets(name, t, ndim_len=None):
    if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor, got {t.dtype} of shape {tuple(t.shape)}")
    if ndim_len is None:
        if t.numel() < 2:
            raise ValueError(f"{name} holds the sequences' ends behind a leading 0: at least two entries")
    elif t.numel() != ndim_len:
        raise ValueError(f"{name} must have {ndim_len} entries, got {t.numel()}")


def packed_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, lengths_k=None, causal=False, scale=None, bias_table=None,
                     buckets=None):
    """softmax(scale q k^T + bias) v within each of the packed sequences.

    q [Tq, H, D] and k, v [Tk, Hkv, D] (fp16 or bf16, contiguous channels,
    any row and head strides) hold the rows of all sequences one behind the
    other; H is a multiple of Hkv and query head h reads key head
    h // (H / Hkv).  D is a multiple of 8 up to 128.  Returns [Tq, H, D].

    ``cu_seqlens_q`` (int32, on the device, [B + 1], from 0) are the row
    offsets of the sequences' queries, ``cu_seqlens_k`` those of their keys
    (the same when left out).  ``lengths_k`` (int32 [B]) says how many of a
    sequence's key rows are in use, for a cache of fixed slots.  Sequences may
    be empty; query rows behind the last sequence come out as 0, as does a
    query that sees no key.

    The last query of a sequence stands at its last key: query i of nq has
    position i + nk - nq.  ``causal`` hides the keys behind that position, and
    one new token per sequence (nq = 1) sees its whole cache.  ``scale`` > 0,
    1 / sqrt(D) by default.

    ``bias_table`` [num_buckets, H] (fp32, fp16 or bf16) with ``buckets``
    (RelativeBuckets) adds table[bucket(key position - query position), head].
    Its gradient is summed in fp32 and returned in the table's type.

    Scores, softmax statistics and sums are fp32; probabilities and their
    gradients are rounded to the input type before each tensor-core product.
    All sums have a fixed order, so equal calls give equal bits.  What lies in
    rows of no sequence, in unused cache rows and in other sequences never
    reaches a result, infinities and NaN included; within a sequence a NaN
    behind the causal mask may reach rows that do not see it.

    Offsets are read on the device and not checked on the host: those that
    decrease or pass the tensors' ends leave the results undefined, touch no
    other memory, and set MN_STATUS_BAD_LENGTHS in attention_status()."""
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError(f"q, k and v must be [rows, heads, head_dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q/k/v must share a dtype")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q/k/v must be float16 or bfloat16, got {q.dtype}")
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    if d < 8 or d > MAX_HEAD_DIM or d % 8:
        raise ValueError(f"head_dim {d} is not supported: a multiple of 8 up to {MAX_HEAD_DIM}")
    if not 1 <= hk <= 65535 or h < 1 or h % hk or h // hk > MAX_GROUP:
        raise ValueError(f"{h} query heads must be a multiple of the {hk} key heads, at most {MAX_GROUP} to one")
    if cu_seqlens_k is None:
        if q.shape[0] != k.shape[0]:
            raise ValueError("without cu_seqlens_k the keys must have the queries' rows")
        cu_seqlens_k = cu_seqlens_q
    _check_offsets("cu_seqlens_q", cu_seqlens_q)
    _check_offsets("cu_seqlens_k", cu_seqlens_k, cu_seqlens_q.numel())
    if lengths_k is not None:
        _check_offsets("lengths_k", lengths_k, cu_seqlens_q.numel() - 1)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if (bias_table is None) != (buckets is None):
        raise ValueError("bias_table and buckets go together")
    if bias_table is not None:
        _check_table(bias_table, buckets, h)
        sides = 2 if buckets.two_sided else 1
        if buckets.num_buckets > MAX_BUCKETS or buckets.num_buckets * (h // hk) > MAX_BIAS_ENTRIES or (sides * buckets.borders[-1] + 1) * (h // hk) > MAX_BIAS_VALUES:
            raise ValueError(f"{buckets} with {h // hk} grouped heads does not fit: at most {MAX_BUCKETS} buckets, "
                             f"{MAX_BIAS_ENTRIES} buckets x grouped heads and {MAX_BIAS_VALUES} distances x grouped heads")
    if max(q.shape[0], k.shape[0]) * max(h // hk, 1) >= 1 << 30:
        raise ValueError("at most 2^30 rows x grouped heads")
    L.require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, lengths_k, bias_table)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (bias_table is not None and bias_table.requires_grad)):
        return _PackedAttention.apply(q, k, v, bias_table, cu_seqlens_q, cu_seqlens_k, lengths_k, bool(causal), scale, buckets)
    return _forward(q, k, v, cu_seqlens_q, cu_seqlens_k, lengths_k, bool(causal), scale, bias_table, buckets, False)[0]


def _bias_forward(table, queries, keys, start, buckets):
    out = torch.empty(table.shape[1], queries, keys, device=table.device, dtype=table.dtype)
    if out.numel():
        t = table.contiguous()
        with torch.cuda.device(table.device):
            L.check(L.lib().mn_relative_bias(table.shape[1], queries, keys, start, buckets.num_buckets, int(buckets.two_sided),
                                             len(buckets.borders), ctypes.addressof(buckets._c_borders), L.dtype_code(t.dtype),
                                             L.ptr(t), L.ptr(out), L.stream_of(t)), "mn_relative_bias")
    return out


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, queries, keys, start, buckets):
        ctx.call = (queries, keys, start, buckets, table.shape[1], table.dtype)
        return _bias_forward(table, queries, keys, start, buckets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dbias):
        queries, keys, start, buckets, heads, dtype = ctx.call
        dev = dbias.device
        d = dbias.contiguous()
        grad = torch.empty(buckets.num_buckets, heads, device=dev, dtype=torch.float32)
        if d.numel() == 0:
            grad.zero_()
        else:
            with torch.cuda.device(dev):
                lib = L.lib()
                nbytes = lib.mn_relative_bias_backward_workspace_bytes(heads, queries, keys, buckets.num_buckets)
                ws = _workspace(nbytes, dev)
                L.check(lib.mn_relative_bias_backward(heads, queries, keys, start, buckets.num_buckets, int(buckets.two_sided),
                                                      len(buckets.borders), ctypes.addressof(buckets._c_borders),
                                                      L.dtype_code(d.dtype), L.ptr(d), L.ptr(grad), L.ptr(ws), nbytes,
                                                      L.stream_of(d)), "mn_relative_bias_backward")
        return grad.to(dtype), None, None, None, None


def relative_position_bias(table, queries, keys, buckets, query_start=None):
    """bias[h, i, j] = table[bucket(j - (i + query_start)), h], [H, queries,
    keys] in the table's type, differentiable in the table [num_buckets, H].

    ``query_start`` is the position of the first query among the keys, by
    default keys - queries (the last query stands at the last key, so a single
    query gets the row of the newest token).  The gradient is summed in fp32
    in a fixed order."""
    _check_table(table, buckets)
    if table.shape[1] < 1:
        raise ValueError("the bias table needs a head")
    if queries < 0 or keys < 0:
        raise ValueError(f"queries and keys must not be negative, got {queries} and {keys}")
    start = keys - queries if query_start is None else operator.index(query_start)
    if max(queries, keys, abs(start)) >= 1 << 30:
        raise ValueError("positions must stay below 2^30")
    L.require_cuda(table)
    if torch.is_grad_enabled() and table.requires_grad:
        return _RelativeBias.apply(table, int(queries), int(keys), start, buckets)
    return _bias_forward(table, int(queries), int(keys), start, buckets)
