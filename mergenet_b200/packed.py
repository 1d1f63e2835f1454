"""Attention over packed sequences of different lengths, and a learned bias
of the relative position by distance buckets.

``packed_attention`` takes the sequences of a batch laid one behind the other
(images of different sizes or numbers of kept tokens, documents, prompts, or one
new token each against a cache) instead of the equal lengths
of ``cross_attention`` and ``local_attention_packed``.  Heads may be grouped,
the mask may be causal, and a learned table adds a bias that depends on the
distance of query and key.  It is differentiable once, in reverse mode, in q,
k, v and the table; forward-mode tangents are refused.

``relative_position_bias`` writes the same bias out as a tensor, for an
attention that takes it as a mask.
"""
from __future__ import annotations

import ctypes
import functools
import operator

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .attention import _STATUS, _status

MAX_HEAD_DIM = 128
MAX_GROUP = 128       # query heads that may share a key head
MAX_BUCKETS = 48      # of a table used inside the attention
MAX_BIAS_GROUP = 16   # query heads that may share a key head then
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

    def __reduce__(self):  # with a module that is saved or sent to another process
        return RelativeBuckets, (self.num_buckets, self.max_distance, self.two_sided)

    def __repr__(self):
        return f"RelativeBuckets({self.num_buckets}, {self.max_distance}, two_sided={self.two_sided})"


def _check_table(table, buckets, heads=None):
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError(f"buckets must be a RelativeBuckets, got {type(buckets).__name__}")
    if table.ndim != 2 or table.shape[0] != buckets.num_buckets or (heads is not None and table.shape[1] != heads):
        want = f"({buckets.num_buckets}, {'heads' if heads is None else heads})"
        raise ValueError(f"the bias table must be {want}, got {tuple(table.shape)}")
    L.dtype_code(table.dtype)


def _ready(t):
    """[rows, heads, channels] with unit channel stride and rows and heads on
    16-byte boundaries (what the copies of a tile need), laid out anew where
    it is not so, a broadcast dimension (stride 0) included."""
    st, sh, sd = t.stride()
    if sd == 1 and not (st % 8 or sh % 8 or t.data_ptr() % 16) and (st > 0 or t.shape[0] < 2) and (sh > 0 or t.shape[1] < 2):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _err_word(dev):
    """The address of the device's status word; none while a graph is being
    captured that would have to create it."""
    st = _STATUS.get((dev.type, dev.index))
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        st = _status(dev)
    return st.data_ptr()


class _on:
    """Makes a device other than the current one current for the launches."""
    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        torch.cuda.set_device(self.before)


def _on_device(dev, fn, *args):
    """fn(*args, stream) with ``dev`` current; stream is its current one."""
    index = dev.index
    if index == torch.cuda.current_device():
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with _on(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def _require(dev, *tensors):
    """All CUDA tensors of one device (the usual case without a loop's cost)."""
    if dev.type == "cuda":
        for t in tensors:
            if t is not None and t.device != dev:
                break
        else:
            return
    L.require_cuda(*tensors)
    raise ValueError("all tensors must be on the same CUDA device")


def _at(t):
    return 0 if t is None else t.data_ptr()


def _args(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, out, lse, dout=None, dq=None, dk=None, dv=None, dbias=None):
    """The bytes of mn_packed_args."""
    tq, h, d = q.shape
    tk, hk, _ = k.shape
    if table is None:
        bias = (0, 0, 0, 0)
        borders = 0
    else:
        bias = (L.dtype_code(table.dtype), buckets.num_buckets, int(buckets.two_sided), len(buckets.borders))
        borders = ctypes.addressof(buckets._c_borders)
    qs, ks, vs, ds = q.stride(), k.stride(), v.stride(), (0, 0) if dout is None else dout.stride()
    return L.PACKED_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), _at(len_k), _at(table),
                              borders, out.data_ptr(), _at(lse), _at(dout), _at(dq), _at(dk), _at(dv), _at(dbias),
                              qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], ds[0], ds[1],
                              cu_q.shape[0] - 1, tq, tk, h, hk, d, L.dtype_code(q.dtype), causal, *bias, scale, 0)


def _launch(fn, size, name, args, dev, stream):
    """Sizes the workspace, allocates it on the current stream and launches."""
    nbytes = size(args)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    rc = fn(args, None if ws is None else ws.data_ptr(), nbytes, _err_word(dev), stream)
    if rc:
        L.check(rc, name)


def _forward(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, want_lse):
    dev = q.device
    q, k, v = _ready(q), _ready(k), _ready(v)
    tq, h, d = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    hk = k.shape[1]
    lse = q.new_empty((hk, tq, h // hk), dtype=torch.float32) if want_lse else None
    if tq:
        table = None if table is None else table.contiguous()
        lib = L.lib()
        _on_device(dev, _launch, lib.mn_packed_attention, lib.mn_packed_attention_workspace_bytes, "mn_packed_attention",
                   _args(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, out, lse), dev)
    return out, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, len_k, causal, scale, buckets):
        out, lse = _forward(q, k, v, cu_q, cu_k, len_k, causal, scale, table, buckets, True)
        ctx.save_for_backward(q, k, v, table, cu_q, cu_k, len_k, out, lse)
        ctx.call = (causal, scale, buckets)
        return out

    @staticmethod
    def backward(ctx, dout):
        return _attention_grads_once(ctx, dout) if torch.is_grad_enabled() else _attention_grads(ctx, dout)


def _attention_grads(ctx, dout):
    q, k, v, table, cu_q, cu_k, len_k, out, lse = ctx.saved_tensors
    causal, scale, buckets = ctx.call
    dev = q.device
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    dbias = None if table is None else torch.empty_like(table, memory_format=torch.contiguous_format)
    if q.numel() == 0:
        for t in (dk, dv, dbias):
            if t is not None:
                t.zero_()
    else:
        tab = None if table is None else table.contiguous()
        q, k, v, dout = _ready(q), _ready(k), _ready(v), _ready(dout)
        lib = L.lib()
        _on_device(dev, _launch, lib.mn_packed_attention_backward, lib.mn_packed_attention_backward_workspace_bytes,
                   "mn_packed_attention_backward",
                   _args(q, k, v, cu_q, cu_k, len_k, causal, scale, tab, buckets, out, lse, dout, dq, dk, dv, dbias), dev)
    return dq, dk, dv, dbias, None, None, None, None, None, None


_attention_grads_once = once_differentiable(_attention_grads)  # where a graph of the gradients is asked for


def _check_sizes(entries, tq, tk, h, hk):
    group = h // hk
    if max(tq, tk) * group >= 1 << 30:
        raise ValueError("at most 2^30 rows x grouped heads")
    if tq * h >= 1 << 31:
        raise ValueError("at most 2^31 query rows x heads")
    if (entries + max(tq // (128 // group), tk // 128)) * hk >= 1 << 31:
        raise ValueError(f"{entries - 1} sequences with {hk} key heads: at most 2^31 tiles of 128 rows x heads, one more a sequence")


def _has_tangent(*tensors):
    """A forward-mode tangent on one of them: the autograd functions have no
    such derivative and refuse the call, where a plain call would drop it."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _check_offsets(name, t, entries):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor, got {t.dtype} of shape {tuple(t.shape)}")
    n = t.shape[0]
    if entries is None:
        if n < 2:
            raise ValueError(f"{name} holds the sequences' ends behind a leading 0: at least two entries")
    elif n != entries:
        raise ValueError(f"{name} must have {entries} entries, got {n}")
    return n


def packed_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, lengths_k=None, causal=False, scale=None, bias_table=None,
                     buckets=None):
    """softmax(scale q k^T + bias) v within each of the packed sequences.

    q [Tq, H, D] and k, v [Tk, Hkv, D] (fp16 or bf16, contiguous channels,
    any row and head strides) hold the rows of all sequences one behind the
    other; H is a multiple of Hkv and query head h reads key head
    h // (H / Hkv).  D is a multiple of 8 up to 128.  Returns [Tq, H, D].
    There are fewer than 2^30 rows x grouped heads, 2^31 query rows x heads and
    2^31 (sequences + tiles of 128 rows) x key heads.

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
    Values beyond +-2^17 ln 2 (90,852) count as that much, a mask's -10^9 or
    lowest value among them; -inf hides its keys outright, and a query that
    sees no others comes out as 0.  The table's gradient is summed in fp32 and
    rounded once to its type.

    Scores, softmax statistics and sums are fp32; probabilities and their
    gradients are rounded to the input type before each tensor-core product
    (in fp16 times a power of two that keeps them in its range, one for each
    sequence and key head).
    All sums have a fixed order, so equal calls give equal bits.  What lies in
    rows of no sequence, in unused cache rows and in other sequences never
    reaches a result, infinities and NaN included; within a sequence a NaN
    behind the causal mask may reach rows that do not see it.

    Offsets are read on the device and not checked on the host: those that
    decrease or pass the tensors' ends leave the results undefined, touch no
    other memory, and set MN_STATUS_BAD_LENGTHS in attention_status(), where it
    stays until reset.  Other calls are not affected."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"q, k and v must be [rows, heads, head_dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    tq, h, d = q.shape
    tk, hk, dk = k.shape
    if (tk, hk, dk) != tuple(v.shape) or d != dk:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    dtype = q.dtype
    if not (dtype == k.dtype == v.dtype):
        raise ValueError("q/k/v must share a dtype")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f"q/k/v must be float16 or bfloat16, got {dtype}")
    if d < 8 or d > MAX_HEAD_DIM or d % 8:
        raise ValueError(f"head_dim {d} is not supported: a multiple of 8 up to {MAX_HEAD_DIM}")
    if not 1 <= hk <= 65535 or h < 1 or h % hk or h // hk > MAX_GROUP:
        raise ValueError(f"{h} query heads must be a multiple of the {hk} key heads, at most {MAX_GROUP} to one")
    group = h // hk
    entries = _check_offsets("cu_seqlens_q", cu_seqlens_q, None)
    if cu_seqlens_k is None:
        if tq != tk:
            raise ValueError("without cu_seqlens_k the keys must have the queries' rows")
        cu_seqlens_k = cu_seqlens_q
    else:
        _check_offsets("cu_seqlens_k", cu_seqlens_k, entries)
    if lengths_k is not None:
        _check_offsets("lengths_k", lengths_k, entries - 1)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -149 <= scale <= 2.0 ** 127:  # in fp32, times log2 e
        raise ValueError(f"scale must be positive and in the range of fp32, got {scale}")
    if (bias_table is None) != (buckets is None):
        raise ValueError("bias_table and buckets go together")
    if bias_table is not None:
        _check_table(bias_table, buckets, h)
        sides = 2 if buckets.two_sided else 1
        if (buckets.num_buckets > MAX_BUCKETS or group > MAX_BIAS_GROUP
                or (sides * buckets.borders[-1] + 1) * group > MAX_BIAS_VALUES):
            raise ValueError(f"{buckets} with {group} grouped heads does not fit: at most {MAX_BUCKETS} buckets, "
                             f"{MAX_BIAS_GROUP} grouped heads and {MAX_BIAS_VALUES} distances x grouped heads")
    if (entries + tq + tk) * h >= 1 << 30:  # smaller ones fit in any case
        _check_sizes(entries, tq, tk, h, hk)
    _require(q.device, q, k, v, cu_seqlens_q, cu_seqlens_k, lengths_k, bias_table)
    causal = bool(causal)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                     or (bias_table is not None and bias_table.requires_grad))) or (
                                         forward_ad._current_level >= 0 and _has_tangent(q, k, v, bias_table)):
        return _PackedAttention.apply(q, k, v, bias_table, cu_seqlens_q, cu_seqlens_k, lengths_k, causal, scale, buckets)
    return _forward(q, k, v, cu_seqlens_q, cu_seqlens_k, lengths_k, causal, scale, bias_table, buckets, False)[0]


def _bias_launch(table, out, queries, keys, start, buckets, stream):
    rc = L.lib().mn_relative_bias(table.shape[1], queries, keys, start, buckets.num_buckets, buckets.two_sided, len(buckets.borders),
                                  ctypes.addressof(buckets._c_borders), L.dtype_code(table.dtype), table.data_ptr(), out.data_ptr(),
                                  stream)
    if rc:
        L.check(rc, "mn_relative_bias")


def _bias_forward(table, queries, keys, start, buckets):
    dev = table.device
    out = torch.empty((table.shape[1], queries, keys), device=dev, dtype=table.dtype)
    if queries and keys:
        _on_device(dev, _bias_launch, table.contiguous(), out, queries, keys, start, buckets)
    return out


def _bias_grad_launch(dbias, grad, start, buckets, stream):
    lib = L.lib()
    heads, queries, keys = dbias.shape
    nb = buckets.num_buckets
    nbytes = lib.mn_relative_bias_backward_workspace_bytes(heads, queries, keys, nb)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dbias.device)
    rc = lib.mn_relative_bias_backward(heads, queries, keys, start, nb, buckets.two_sided, len(buckets.borders),
                                       ctypes.addressof(buckets._c_borders), L.dtype_code(dbias.dtype), dbias.data_ptr(),
                                       grad.data_ptr(), ws.data_ptr(), nbytes, stream)
    if rc:
        L.check(rc, "mn_relative_bias_backward")


def _bias_grads(ctx, dbias):
    start, buckets = ctx.call
    grad = torch.empty((buckets.num_buckets, dbias.shape[0]), device=dbias.device, dtype=dbias.dtype)
    if dbias.numel():
        _on_device(dbias.device, _bias_grad_launch, dbias.contiguous(), grad, start, buckets)
    else:
        grad.zero_()
    return grad, None, None, None, None


_bias_grads_once = once_differentiable(_bias_grads)


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, queries, keys, start, buckets):
        ctx.call = (start, buckets)
        return _bias_forward(table, queries, keys, start, buckets)

    @staticmethod
    def backward(ctx, dbias):
        return _bias_grads_once(ctx, dbias) if torch.is_grad_enabled() else _bias_grads(ctx, dbias)


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
    queries, keys = operator.index(queries), operator.index(keys)
    if queries < 0 or keys < 0:
        raise ValueError(f"queries and keys must not be negative, got {queries} and {keys}")
    start = keys - queries if query_start is None else operator.index(query_start)
    if queries + keys + abs(start) >= 1 << 30:
        raise ValueError("positions and distances must stay below 2^30")
    if table.shape[1] > 65535 or queries > 32 * 65535:
        raise ValueError("at most 65535 heads and 2097120 queries")
    L.require_cuda(table)
    if (torch.is_grad_enabled() and table.requires_grad) or (forward_ad._current_level >= 0 and _has_tangent(table)):
        return _RelativeBias.apply(table, queries, keys, start, buckets)
    return _bias_forward(table, queries, keys, start, buckets)
