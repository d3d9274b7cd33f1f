"""What the operators over a paged cache refuse, without a GPU: every call here is turned down before a device is asked for."""
import ctypes as C

import pytest
import torch

from glinthawk_amd import Shape, _lib, ops

AT = 1 << 20          # an address that nothing reads
SHAPE = Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=2, hidden_dim=8, seq_len=8)
ROW = 2 * SHAPE.kv_dim


def pages(dt_size=2, **other):
    p = _lib.GhPages(AT, 16 * ROW * dt_size, 10, 16, AT, 4)
    for name, value in other.items():
        setattr(p, name, value)
    return p


def shape(**other):
    s = SHAPE.c()
    for name, value in other.items():
        setattr(s, name, value)
    return s


def decode(p=None, s=None, q=AT, out=AT * 2, lengths=AT, batch=3, most=64, dt=0):
    return _lib.lib().gh_attn_decode_paged(q, C.byref(p or pages()), lengths, out, batch, most, C.byref(s or shape()), dt, None, 0, None)


def packed(p=None, s=None, q=AT, out=AT * 2, first=AT, batch=3, tokens=30, most=64, dt=0):
    return _lib.lib().gh_attn_packed(q, C.byref(p or pages()), first, None, out, batch, tokens, most, C.byref(s or shape()), dt, None, 0, None)


def rows(p=None, first=AT, batch=3, tokens=30, kv=SHAPE.kv_dim, dt=0):
    return _lib.lib().gh_page_rows(C.byref(p or pages()), first, None, batch, tokens, kv, AT, AT, dt, None)


def refused(rc, said):
    text = _lib.lib().gh_last_error().decode()
    assert rc == -1 and said in text, (rc, text)


@pytest.mark.parametrize("call", [decode, packed, rows])
@pytest.mark.parametrize("what,said", [
    (dict(pool=None), "NULL"), (dict(table=None), "NULL"), (dict(n_pages=0), "no pages"), (dict(table_stride=0), "no pages"), (dict(page_tokens=0), "power of two"),
    (dict(page_tokens=24), "power of two"), (dict(page_tokens=1 << 22), "2 GiB"), (dict(page_stride=16 * ROW * 2 - 2), "apart"), (dict(page_stride=16 * ROW * 2 + 1), "apart"),
    (dict(page_stride=1 << 40), "apart"), (dict(pool=AT + 1), "aligned"), (dict(table=AT + 2), "aligned"), (dict(table_stride=1 << 27), "2^31")])
def test_pages_that_are_refused(call, what, said):
    refused(call(pages(**what)), said)


@pytest.mark.parametrize("call", [decode, packed])
@pytest.mark.parametrize("what,said", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(dt=3), "dtype"), (dict(dt=-1), "dtype"), (dict(most=65), "reaches"), (dict(q=AT + 1), "aligned"), (dict(out=AT + 1), "aligned"),
    (dict(out=AT + 2), "over q"), (dict(batch=(1 << 20) + 1), "too many"), (dict(s=shape(head_size=0)), "shape"), (dict(s=shape(head_size=257)), "shape"), (dict(s=shape(gqa_size=3)), "shape"),
    (dict(s=shape(kv_dim=512)), "shape"), (dict(s=shape(n_kv_heads=0)), "shape"), (dict(p=pages(page_stride=16 * ROW * 2), dt=1), "apart")])
def test_attention_that_is_refused(call, what, said):
    refused(call(**what), said)


def test_tables_that_are_refused():
    refused(decode(lengths=None), "NULL")
    refused(packed(first=None), "NULL")
    refused(packed(tokens=(1 << 24) + 1), "too many")
    refused(rows(first=None), "NULL")
    refused(rows(kv=0), "kv_dim")
    refused(rows(dt=5), "dtype")
    refused(rows(batch=0), "shape")


def copy(pairs, n_pages=8, stride=64, size=64, layers=1, layer_stride=0, pool=AT):
    flat = [v for p in pairs for v in p]
    return _lib.lib().gh_copy_pages_host(pool, stride, size, n_pages, layers, layer_stride, (C.c_uint32 * max(1, len(flat)))(*flat), len(pairs), None)


def test_copies_that_are_refused():
    refused(copy([(0, 1)], pool=None), "NULL")
    refused(copy([(0, 8)]), "of 8 pages")
    refused(copy([(8, 0)]), "of 8 pages")
    refused(copy([(0, 1), (2, 1)]), "page 1 is written twice")
    refused(copy([(0, 1), (1, 2)]), "page 1 is read and written")
    refused(copy([(3, 3)]), "page 3 is read and written")
    refused(copy([(0, 1)], stride=32), "bad pages")
    refused(copy([(0, 1)], size=0), "bad pages")
    refused(copy([(0, 1)], n_pages=0), "bad pages")
    refused(copy([(0, 1)], layers=2, layer_stride=64), "layers")          # a layer inside the other's pages
    refused(copy([(0, 1)], layers=70000, layer_stride=1024), "layers")
    assert _lib.lib().gh_copy_pages(AT, 64, 64, 8, 1, 0, None, 3, None) == -1
    assert _lib.lib().gh_copy_pages(AT, 64, 64, 8, 1, 0, AT + 2, 3, None) == -1


def logprobs(given=AT, entropy=AT, ids=AT, values=AT, logits=AT, stride=100, tokens=AT, vocab=100, n_rows=2, top=3, dt=1):
    return _lib.lib().gh_token_logprobs(given, entropy, ids, values, logits, stride, tokens, vocab, n_rows, top, dt, None, 0, None)


@pytest.mark.parametrize("what,said", [
    (dict(logits=None), "NULL"), (dict(tokens=None), "NULL"), (dict(ids=None), "NULL"), (dict(values=None), "NULL"), (dict(dt=4), "dtype"), (dict(vocab=0), "shape"),
    (dict(vocab=(1 << 21) + 1, stride=1 << 22), "shape"), (dict(n_rows=65536), "shape"), (dict(top=65), "alternatives"), (dict(top=3, vocab=2), "alternatives"), (dict(stride=99), "apart"),
    (dict(logits=AT + 2), "aligned")])
def test_logits_that_are_refused(what, said):
    refused(logprobs(**what), said)


def test_tensors_that_are_refused():
    """What the tensor front end turns down by itself."""
    pool, table = torch.zeros(4, 16, ROW, dtype=torch.float16), torch.zeros((2, 3), dtype=torch.int32)
    for bad in (pool[0], pool.transpose(1, 2), pool[:, :, ::2], pool[:, ::2]):
        with pytest.raises(ValueError):
            ops.pages(bad, table)
    for bad in (table[0], table.long(), table.t()):
        with pytest.raises(ValueError):
            ops.pages(pool, bad)
    p = ops.pages(pool, table)
    q, lengths, first = torch.zeros(2, 1024, dtype=torch.float16), torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    good = dict(q=q, lengths=lengths, xb=q.clone(), shape=SHAPE)
    for bad in (dict(q=q.float()), dict(q=q[:, :1000]), dict(q=q[:1]), dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(xb=q[:1].clone()), dict(xb=q.float()),
                dict(shape=Shape(dim=1024, n_layers=1, n_heads=8, n_kv_heads=4, hidden_dim=8, seq_len=8)), dict(q=torch.zeros(3, 1024, dtype=torch.float16), lengths=torch.ones(3, dtype=torch.int32)),
                dict(q=q.to("meta"))):
        a = dict(good, **bad)
        with pytest.raises(ValueError):
            ops.attn_decode_paged(a["q"], p, a["lengths"], a["xb"], 16, a["shape"], torch.zeros(16, dtype=torch.uint8))
    for bad in (dict(first=first.long()), dict(start=lengths.long()), dict(start=lengths[:1]), dict(first=torch.zeros(4, dtype=torch.int32), start=None)):
        a = dict(dict(first=first, start=lengths), **bad)
        with pytest.raises(ValueError):
            ops.attn_packed(q, p, a["first"], a["start"], q.clone(), 16, SHAPE, torch.zeros(16, dtype=torch.uint8))
        with pytest.raises(ValueError):
            ops.page_rows(p, a["first"], a["start"], 2)
    with pytest.raises(ValueError):
        ops.copy_pages(pool, torch.zeros((2, 3), dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.copy_pages(pool, torch.zeros((2, 2), dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.copy_pages(pool[:, ::2], [(0, 1)])
    for pairs in ([(0, 2 ** 32 + 1)], [(0, -1)], [(0, pool.shape[0])], [(0, 1, 2), (3, 0, 1)]):
        with pytest.raises(ValueError):
            ops.copy_pages(pool, pairs)
    for logits, tokens in ((torch.zeros(2, 9), lengths.long()), (torch.zeros(2, 9), lengths[:1]), (torch.zeros(9, 2).t(), lengths), (torch.zeros(9), lengths)):
        with pytest.raises(ValueError):
            ops.token_logprobs(logits, tokens, 1, torch.zeros(16, dtype=torch.uint8))


def test_what_a_call_of_nothing_says_without_a_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert decode(batch=0) == -3 and packed(tokens=0) == -3 and copy([]) == -3 and logprobs(n_rows=0) == -3      # nothing works without a device


def test_workspaces_cover_smaller_calls():
    """A workspace made for the largest batch and length serves every smaller call."""
    s = shape()
    L = _lib.lib()
    for most in (1, 64, 300, 5000, 40000):
        assert L.gh_attn_decode_paged_workspace(0, most, C.byref(s), 0) == 0 and L.gh_attn_packed_workspace(0, 5, most, C.byref(s), 0) == 0
    assert L.gh_token_logprobs_workspace(0, 5, 1) == 0 and L.gh_token_logprobs_workspace(1, 100, 5) == 0
