"""Refusals of the serving operators: everything the host can see is checked before any device work, so these run without a GPU."""
import ctypes as C

import pytest
import torch

import puppygrad_b200 as pg
from puppygrad_b200 import _native as N

P = 1 << 20  # stands for a device address: never dereferenced


def cache(**kw):
    c = N.PgKv8Cache(pool=P, scales=P, page_table=P, n_pages=4, page_tokens=16, kv_heads=2, head_dim=64, seqs=3, pages_per_seq=5, device=0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append(c=None, k=P, ks=128, v=P, vs=128, q=0, qs=0, o=0, os=0, dtype=0, heads=0, rows=3, start=0, lens=P, rot=0, base=1e4):
    return N.lib.pg_kv8_append(C.byref(c or cache()), k, ks, v, vs, q, qs, o, os, dtype, heads, rows, start, lens, rot, base, 0)


def attention(c=None, q=P, qs=256, o=P, os=256, dtype=0, heads=4, rows=3, most=1, start=0, lens=P, scale=0.125, window=0, keep=0, ws=P, size=1 << 40):
    return N.lib.pg_kv8_attention(C.byref(c or cache()), q, qs, o, os, dtype, heads, rows, most, start, lens, scale, window, keep, ws, size, 0)


def linear(x=P, xs=64, p=P, s=P, b=0, dtype=0, m=1, n=16, k=64, group=64, o=P, os=16):
    return N.lib.pg_linear_q4(x, xs, p, s, b, dtype, m, n, k, group, o, os, 0, 0)


def logprobs(x=P, xs=100, dtype=0, rows=2, vocab=100, t=P, lp=P, e=P, k=0, ids=0, values=0):
    return N.lib.pg_token_logprobs(x, xs, dtype, rows, vocab, t, lp, e, k, ids, values, 0, 0)


def refused(status, text):
    assert status == N.PG_INVALID_INPUT
    assert text in N.lib.pg_last_error_message().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(pool=0), "null pool"), (dict(scales=0), "null pool"), (dict(page_table=0), "null pool"), (dict(pool=P + 8), "16-byte aligned"),
    (dict(scales=P + 4), "not aligned"), (dict(n_pages=0), "n_pages"), (dict(page_tokens=48), "page_tokens 48 must be 16, 32 or 64"), (dict(kv_heads=0), "kv_heads 0"),
    (dict(head_dim=63), "head_dim 63 must be even"), (dict(head_dim=258), "head_dim 258"), (dict(head_dim=0), "head_dim 0"), (dict(seqs=0), "seqs 0"),
    (dict(seqs=4097), "seqs 4097"), (dict(pages_per_seq=0), "pages_per_seq 0"), (dict(pages_per_seq=1 << 27), "2^30"),
])
def test_cache_is_checked(kw, text):
    refused(append(cache(**kw)), text)
    refused(attention(cache(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(k=0), "k is null"), (dict(v=0), "v is null"), (dict(ks=127), "k: distance between rows 127 is less than a row of 128"), (dict(vs=0), "v: distance"),
    (dict(dtype=2), "dtype 2"), (dict(lens=0), "lens is null"), (dict(rows=4), "must be seqs 3"), (dict(rows=-1, start=P), "rows must not be negative"),
    (dict(rot=3), "rot_dims 3"), (dict(rot=66), "rot_dims 66"), (dict(rot=-2), "rot_dims -2"), (dict(rot=2, base=0.0), "rot_base"),
    (dict(rot=2, base=float("nan")), "rot_base"), (dict(q=P), "given together"), (dict(o=P), "given together"), (dict(q=P, o=P, heads=3, qs=192, os=192), "heads 3"),
    (dict(q=P, o=P, heads=4, qs=255, os=256), "q: distance"), (dict(q=P, o=P, heads=4, qs=256, os=300), "in place"), (dict(k=P + 2), "k is not aligned"),
    (dict(rows=1 << 30, start=P, c=cache(kv_heads=1024), ks=1 << 20, vs=1 << 20), "too many"),
])
def test_append_is_checked(kw, text):
    refused(append(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=0), "q is null"), (dict(o=0), "out is null"), (dict(heads=5), "heads 5 must be 1 to 128 times kv_heads 2"), (dict(heads=0), "heads 0"),
    (dict(heads=512), "heads 512"), (dict(qs=255), "q: distance"), (dict(os=255), "out: distance"), (dict(scale=float("inf")), "scale"), (dict(window=-1), "window"),
    (dict(keep=-1), "window"), (dict(most=0), "max_rows"), (dict(ws=0), "workspace of 0 bytes"), (dict(size=100), "workspace of 100 bytes"),
    (dict(ws=P + 128), "256-byte aligned"), (dict(dtype=7), "dtype 7"), (dict(rows=2), "must be seqs 3"),
    (dict(rows=1 << 28, start=P, c=cache(pages_per_seq=1 << 20)), "too many for one call"),
])
def test_attention_is_checked(kw, text):
    refused(attention(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(m=0), "m 0 must be in 1..16"), (dict(m=17), "m 17"), (dict(n=0), "n and k"), (dict(k=0), "n and k"), (dict(group=32), "group 32"), (dict(p=0), "packed or scales"),
    (dict(s=0), "packed or scales"), (dict(p=P + 8), "16-byte aligned"), (dict(s=P + 8), "16-byte aligned"), (dict(xs=63), "x: distance"), (dict(os=15), "out: distance"), (dict(dtype=-1), "dtype -1"),
    (dict(b=P + 2), "bias"), (dict(x=P + 1, dtype=1), "x is not aligned"),
])
def test_linear_q4_is_checked(kw, text):
    refused(linear(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(x=0), "logits is null"), (dict(vocab=0), "vocab 0"), (dict(xs=99), "logits: distance"), (dict(t=0), "given together"), (dict(lp=0), "given together"),
    (dict(k=33, ids=P, values=P), "top_k 33"), (dict(k=101, ids=P, values=P), "top_k 101"), (dict(k=2, ids=P), "top_ids or top_logprobs"), (dict(k=-1), "top_k -1"),
    (dict(t=0, lp=0, e=0), "no output"), (dict(rows=-1), "rows"), (dict(e=P + 2), "aligned"), (dict(vocab=5, xs=5, k=6, ids=P, values=P), "top_k 6"),
])
def test_token_logprobs_is_checked(kw, text):
    refused(logprobs(**kw), text)


def test_rows_of_all_heads_are_numbered_with_31_bits():
    refused(attention(rows=1 << 30, start=P, heads=4), "too many for one call")


def test_calls_without_rows_do_nothing():
    assert append(rows=0, start=P) == N.PG_OK and attention(rows=0, start=P) == N.PG_OK and logprobs(rows=0) == N.PG_OK


def test_sizes():
    assert N.lib.pg_kv8_pool_bytes(10, 16, 2, 64) == 10 * 2 * 2 * 16 * 64
    assert N.lib.pg_kv8_pool_bytes(10, 16, 2, 65) == 0 and N.lib.pg_kv8_pool_bytes(1, 64, 1, 66) == 2 * 64 * 128
    assert N.lib.pg_q4_packed_bytes(17, 65) == 2 * 2 * 512 and N.lib.pg_q4_scale_bytes(17, 65, 64) == 2 * 32 * 2
    assert N.lib.pg_q4_packed_bytes(0, 1) == 0 and N.lib.pg_q4_scale_bytes(1, 1, 16) == 0
    assert pg.q4_shapes(17, 200, 128) == ((2, 4, 512), (2, 32))
    assert pg.Kv8Cache.pool_shape(3, 2, 32, 96) == (3, 2, 2 * 32 * 128)
    with pytest.raises(pg.Gpt2Error, match="page_tokens 8"):
        pg.Kv8Cache.pool_shape(3, 2, 8, 96)
    with pytest.raises(pg.Gpt2Error, match="group 100"):
        pg.q4_shapes(17, 200, 100)


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 100)
    with pytest.raises(pg.Gpt2Error, match="a CUDA device is needed"):
        pg.token_logprobs(x, entropy=torch.zeros(2))
    with pytest.raises(pg.Gpt2Error, match="a CUDA device is needed"):
        pg.linear_q4(x, x, x, x, 64)
    with pytest.raises(pg.Gpt2Error, match="dtype torch.float64"):
        pg.token_logprobs(x.double(), entropy=torch.zeros(2))
    with pytest.raises(pg.Gpt2Error, match="a CUDA device is needed"):
        pg.Kv8Cache(x, x, x, page_tokens=16, head_dim=64)


def test_buffers_with_another_number_of_dimensions_are_refused():
    x, y = torch.zeros(5), torch.zeros(2, 5)
    for call in (lambda: pg.token_logprobs(x), lambda: pg.linear_q4(x, y, y, y, 64), lambda: pg.linear_q4(y, y, y, x, 64), lambda: pg.quantize_q4(x, y, y, 64)):
        with pytest.raises(pg.Gpt2Error, match=r"\(5,\) must have 2 dimensions"):
            call()


class Buffer:
    """What the operators look at of a tensor on a device; its address is never used by a call that is refused."""

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, "cuda:0"

    def stride(self):
        return tuple(torch.empty(self.shape, device="meta").stride())

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def data_ptr(self):
        return P


def int32(*shape):
    return Buffer(*shape, dtype=torch.int32)


@pytest.mark.parametrize("far", [1 << 31, (1 << 32) + 1, -1])
def test_numbers_beyond_32_bits_are_refused(far):
    """They would be taken modulo 2^32: a window of 2^32 for none at all, 2^32 rows for no rows."""
    handle = pg.Kv8Cache(Buffer(4, 2, 2 * 16 * 64, dtype=torch.uint8), Buffer(4, 2, 2), int32(3, 5), page_tokens=16, head_dim=64)
    q, k, lens, ws = Buffer(3, 4, 64), Buffer(3, 2, 64), int32(3), Buffer(1 << 30, dtype=torch.uint8)
    calls = [lambda: handle.attention(q, q, lens, ws, window=far), lambda: handle.attention(q, q, lens, ws, keep_first=far),
             lambda: handle.attention(q, q, lens, ws, row_start=int32(4), max_rows=far), lambda: handle.append(k, k, lens, rot_dims=far),
             lambda: handle.workspace_bytes(far, 4, torch.float32), lambda: handle.workspace_bytes(3, far, torch.float32),
             lambda: pg.q4_shapes(far, 64, 64), lambda: pg.q4_shapes(64, far, 64), lambda: pg.q4_shapes(64, 64, far), lambda: pg.Kv8Cache.pool_shape(far, 2, 16, 64),
             lambda: pg.Kv8Cache.pool_shape(4, 2, 16, far), lambda: pg.linear_q4(Buffer(1, 64), Buffer(1, 1, 512, dtype=torch.uint8), Buffer(1, 16, dtype=torch.bfloat16), Buffer(1, 16), far)]
    if far > 0:
        calls += [lambda: pg.token_logprobs(Buffer(far, 1), entropy=Buffer(far)), lambda: pg.token_logprobs(Buffer(1, far), entropy=Buffer(1)),
                  lambda: pg.token_logprobs(Buffer(1, 100), top_ids=int32(1, far), top_logprobs=Buffer(1, far)), lambda: handle.append(Buffer(far, 2, 64), Buffer(far, 2, 64), lens, row_start=int32(4)),
                  lambda: pg.Kv8Cache(Buffer(4, 2, 2 * 16 * 64, dtype=torch.uint8), Buffer(4, 2, 2), int32(1, far), page_tokens=16, head_dim=64)]
    for call in calls:
        with pytest.raises(pg.Gpt2Error, match=f"{far} must be in 0..2\\^31-1"):
            call()
