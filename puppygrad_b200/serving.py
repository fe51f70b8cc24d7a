"""Operators of a serving program on its own device buffers: a paged cache of keys and values in 8 bits, products with 4-bit weights, log
probabilities of given tokens. include/puppygrad_b200.h has the layouts and what each call promises.

Buffers are anything with the interface of a torch tensor (`data_ptr`, `shape`, `stride`, `is_contiguous`, `dtype`, `get_device`); torch
itself is not imported. Calls are enqueued on `stream` (a CUDA stream's address, 0 = the default stream) and return without waiting; what they
read must stay allocated until they have run.
"""
from __future__ import annotations

import ctypes as C
from typing import Any, Dict, Optional, Tuple

from . import _native as N
from .errors import Gpt2Error, check

_CODES = {"torch.float32": 0, "torch.bfloat16": 1}
_seen: Dict[Any, Optional[str]] = {}  # names of dtype objects: printing one takes longer than all of a tensor's other checks


def _name(dtype) -> str:
    name = _seen.get(dtype)
    if name is None:
        name = _seen[dtype] = str(dtype)
    return name


def _bad(what: str):
    return Gpt2Error("InvalidInput", what)


def _checked(**numbers: int) -> None:
    """The library takes these as 32 bits and would not see what is beyond. (Calls of a step "or" the numbers together first, which is quicker.)"""
    for name, n in numbers.items():
        if n >> 31:
            raise _bad(f"{name} {n} must be in 0..2^31-1")


def _code(t, name: str) -> int:
    code = _CODES.get(_name(t.dtype))
    if code is None:
        raise _bad(f"{name}: dtype {t.dtype} must be float32 or bfloat16")
    return code


def _device(t, name: str) -> int:
    device = t.get_device()
    if device < 0:
        raise _bad(f"{name} is on {t.device}, a CUDA device is needed")
    return device


def _sides(t, name: str, n: int):
    """Shape of a buffer that has to have n dimensions."""
    if len(t.shape) != n:
        raise _bad(f"{name} {tuple(t.shape)} must have {n} dimensions")
    return t.shape


def _flat(t, name: str, dtype: str, shape: Tuple[int, ...], device: int) -> int:
    """Address of a buffer that has to be contiguous and of that type and shape."""
    if t.shape == shape and _seen.get(t.dtype) == dtype and t.is_contiguous() and t.get_device() == device:
        return t.data_ptr()
    if t.shape != shape or _name(t.dtype) != dtype or not t.is_contiguous():
        raise _bad(f"{name}: {dtype} {shape} without gaps is needed, got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    if t.get_device() != device:
        raise _bad(f"{name} is on {t.device}, the others are on cuda:{device}")
    return t.data_ptr()


def _rows(t, name: str, dtype, shape: Tuple[int, ...], device: int) -> Tuple[int, int]:
    """Address and distance between rows of a buffer of that type and shape, whose rows are without gaps."""
    if t.shape != shape or t.dtype != dtype:
        raise _bad(f"{name}: {dtype} {shape} is needed, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device:
        raise _bad(f"{name} is on {t.device}, the others are on cuda:{device}")
    stride, width = t.stride(), shape[-1]
    gap = stride[-1] != 1 and width > 1
    if len(shape) == 3:
        gap = gap or (stride[1] != width and shape[1] > 1)
        width *= shape[1]
    if gap:
        raise _bad(f"{name}: a row must be without gaps, got strides {stride}")
    # of a single row (or none) the distance says nothing
    return t.data_ptr(), stride[0] if shape[0] > 1 else width


class Kv8Cache:
    """One layer's keys and values in 8 bits, in buffers of the caller: `pool` uint8 [n_pages, kv_heads, 2 * page_tokens * padded] with
    padded = head_dim rounded up to 64, `scales` float32 [n_pages, kv_heads, 2], `page_table` int32 [seqs, pages_per_seq]. The object
    holds references to them and nothing of their contents: pages are handed out by writing page_table."""

    def __init__(self, pool, scales, page_table, page_tokens: int, head_dim: int):
        device = _device(pool, "pool")
        seqs, per_seq = _sides(page_table, "page_table", 2)
        _checked(seqs=seqs, pages_per_seq=per_seq)
        n_pages, kv_heads = _sides(pool, "pool", 3)[:2]
        self._c = N.PgKv8Cache()
        self._c.pool = _flat(pool, "pool", "torch.uint8", self.pool_shape(n_pages, kv_heads, page_tokens, head_dim), device)
        self._c.scales = _flat(scales, "scales", "torch.float32", (n_pages, kv_heads, 2), device)
        self._c.page_table = _flat(page_table, "page_table", "torch.int32", tuple(page_table.shape), device)
        self._c.n_pages, self._c.page_tokens, self._c.kv_heads, self._c.head_dim = n_pages, page_tokens, kv_heads, head_dim
        self._c.seqs, self._c.pages_per_seq, self._c.device = page_table.shape[0], page_table.shape[1], device
        self.pool, self.scales, self.page_table = pool, scales, page_table
        self.kv_heads, self.head_dim, self.seqs, self.device = kv_heads, head_dim, page_table.shape[0], device
        self._ref = C.byref(self._c)

    @staticmethod
    def pool_shape(n_pages: int, kv_heads: int, page_tokens: int, head_dim: int) -> Tuple[int, int, int]:
        _checked(n_pages=n_pages, kv_heads=kv_heads, page_tokens=page_tokens, head_dim=head_dim)
        size = N.lib.pg_kv8_pool_bytes(n_pages, page_tokens, kv_heads, head_dim)
        if not size:
            raise _bad(N.lib.pg_last_error_message().decode())
        return n_pages, kv_heads, size // (n_pages * kv_heads)

    def append(self, k, v, lens, row_start=None, q=None, q_out=None, rot_dims: int = 0, rot_base: float = 10000.0, stream: int = 0) -> None:
        """Appends k and v [rows, kv_heads, head_dim], k turned by its positions; q [rows, heads, head_dim] is turned into q_out (which
        may be q). Sequence b has rows row_start[b] : row_start[b + 1] (None: row b), at the last positions of lens[b], its
        length with them."""
        rows, device, kind = _sides(k, "k", 3)[0], self.device, k.dtype
        dtype, shape = _code(k, "k"), (rows, self.kv_heads, self.head_dim)
        kp, ks = _rows(k, "k", kind, shape, device)
        vp, vs = _rows(v, "v", kind, shape, device)
        qp = qs = op = os = heads = 0
        if q is not None or q_out is not None:
            if q is None or q_out is None:
                raise _bad("q and q_out must be given together")
            heads = _sides(q, "q", 3)[1]
            shape = (rows, heads, self.head_dim)
            qp, qs = _rows(q, "q", kind, shape, device)
            op, os = _rows(q_out, "q_out", kind, shape, device)
        if (rows | heads | rot_dims) >> 31:
            _checked(rows=rows, heads=heads, rot_dims=rot_dims)
        lp = _flat(lens, "lens", "torch.int32", (self.seqs,), device)
        sp = 0 if row_start is None else _flat(row_start, "row_start", "torch.int32", (self.seqs + 1,), device)
        status = N.lib.pg_kv8_append(self._ref, kp, ks, vp, vs, qp, qs, op, os, dtype, heads, rows, sp, lp, rot_dims, rot_base, stream)
        if status:
            check(status)

    def workspace_bytes(self, rows: int, heads: int, dtype) -> int:
        """Size of the workspace of `attention` calls of up to that many rows; its memory must be zero before its first use. Calls over
        different caches, rows and heads can share one, one after the other, if it has the most bytes that any of them needs."""
        _checked(rows=rows, heads=heads)
        code = _CODES.get(_name(dtype), -1)
        size = N.lib.pg_kv8_attention_workspace_bytes(self._ref, rows, heads, code)
        if not size:
            raise _bad(N.lib.pg_last_error_message().decode())
        return size

    def attention(self, q, out, lens, workspace, row_start=None, max_rows: int = 1, scale: Optional[float] = None, window: int = 0,
                  keep_first: int = 0, stream: int = 0) -> None:
        """out = softmax(scale * q . k) v over what each row sees; q and out [rows, heads, head_dim], scale head_dim ** -0.5 unless
        given, `lens` and `row_start` as in `append`. max_rows: at least the rows of any sequence. `workspace`: uint8, zeroed
        before its first use, of workspace_bytes(); calls that may overlap on the GPU need one each. Its first 4 bytes stay zero
        unless a wait within a kernel ran out, which leaves NaN rows."""
        device, kind, shape = self.device, q.dtype, (*_sides(q, "q", 3)[:2], self.head_dim)
        rows, heads = shape[:2]
        if (rows | heads | max_rows | window | keep_first) >> 31:
            _checked(rows=rows, heads=heads, max_rows=max_rows, window=window, keep_first=keep_first)
        dtype = _code(q, "q")
        qp, qs = _rows(q, "q", kind, shape, device)
        op, os = _rows(out, "out", kind, shape, device)
        lp = _flat(lens, "lens", "torch.int32", (self.seqs,), device)
        sp = 0 if row_start is None else _flat(row_start, "row_start", "torch.int32", (self.seqs + 1,), device)
        size = _sides(workspace, "workspace", 1)[0]
        wp = _flat(workspace, "workspace", "torch.uint8", (size,), device)
        status = N.lib.pg_kv8_attention(self._ref, qp, qs, op, os, dtype, heads, rows, max_rows, sp, lp,
                                        self.head_dim ** -0.5 if scale is None else scale, window, keep_first, wp, size, stream)
        if status:
            check(status)


def q4_shapes(n: int, k: int, group: int) -> Tuple[Tuple[int, int, int], Tuple[int, int]]:
    """Shapes of the packed codes (uint8) and the scales (bfloat16) of a 4-bit matrix of n outputs and k inputs."""
    _checked(n=n, k=k, group=group)
    if not N.lib.pg_q4_scale_bytes(n, k, group):
        raise _bad(N.lib.pg_last_error_message().decode())
    return (-(-n // 16), -(-k // 64), 512), (-(-k // group), -(-n // 16) * 16)


def quantize_q4(w, packed, scales, group: int, stream: int = 0) -> None:
    """Lays the matrix w [n, k] out in 4 bits, with one scale for every `group` (64 or 128) inputs of an output."""
    n, k = _sides(w, "w", 2)
    dtype, device = _code(w, "w"), _device(w, "w")
    wp, ws = _rows(w, "w", w.dtype, (n, k), device)
    ps, ss = q4_shapes(n, k, group)
    check(N.lib.pg_quantize_q4(wp, ws, dtype, n, k, group, _flat(packed, "packed", "torch.uint8", ps, device),
                               _flat(scales, "scales", "torch.bfloat16", ss, device), device, stream))


def linear_q4(x, packed, scales, out, group: int, bias=None, stream: int = 0) -> None:
    """out [m, n] = x [m, k] @ dequant(w [n, k]).T + bias for up to 16 rows."""
    m, k = _sides(x, "x", 2)
    n, kind = _sides(out, "out", 2)[1], x.dtype
    if (m | n | k | group) >> 31:
        _checked(m=m, n=n, k=k, group=group)
    dtype, device = _code(x, "x"), _device(x, "x")
    xp, xs = _rows(x, "x", kind, (m, k), device)
    op, os = _rows(out, "out", kind, (m, n), device)
    tiles = -(-n // 16)
    pp = _flat(packed, "packed", "torch.uint8", (tiles, -(-k // 64), 512), device)
    sp = _flat(scales, "scales", "torch.bfloat16", (-(-k // group) if group > 0 else 0, tiles * 16), device)
    bp = 0 if bias is None else _flat(bias, "bias", _name(kind), (n,), device)
    status = N.lib.pg_linear_q4(xp, xs, pp, sp, bp, dtype, m, n, k, group, op, os, device, stream)
    if status:
        check(status)


def token_logprobs(logits, targets=None, logprobs=None, entropy=None, top_ids=None, top_logprobs=None, stream: int = 0) -> None:
    """Scores of the rows of logits [rows, vocab]: logprobs [rows] of `targets` [rows], entropy [rows], the most likely ids and their
    log probabilities [rows, k] (k up to 32), each where its output is given."""
    rows, vocab = _sides(logits, "logits", 2)
    if (rows | vocab) >> 31:
        _checked(rows=rows, vocab=vocab)
    dtype, device, each = _code(logits, "logits"), _device(logits, "logits"), (rows,)
    lp, ls = _rows(logits, "logits", logits.dtype, (rows, vocab), device)
    if (top_ids is None) != (top_logprobs is None):
        raise _bad("top_ids and top_logprobs must be given together")
    tp = 0 if targets is None else _flat(targets, "targets", "torch.int32", each, device)
    op = 0 if logprobs is None else _flat(logprobs, "logprobs", "torch.float32", each, device)
    ep = 0 if entropy is None else _flat(entropy, "entropy", "torch.float32", each, device)
    k = ip = vp = 0
    if top_ids is not None:
        k = _sides(top_ids, "top_ids", 2)[1]
        _checked(top_k=k)
        ip = _flat(top_ids, "top_ids", "torch.int32", (rows, k), device)
        vp = _flat(top_logprobs, "top_logprobs", "torch.float32", (rows, k), device)
    status = N.lib.pg_token_logprobs(lp, ls, dtype, rows, vocab, tp, op, ep, k, ip, vp, device, stream)
    if status:
        check(status)
