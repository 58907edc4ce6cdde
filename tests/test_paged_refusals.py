"""CPU: what the paged cache's calls refuse before they touch a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from blockedattention_b200 import _lib as L
from blockedattention_b200 import blockPagedAppend, blockPagedAttention, blockPagedSlots

P = 1 << 20  # an aligned address that no call here gets as far as reading


def cache(**kw):
    base = dict(k=P, v=P, pages=8, page_size=16, heads=4, head_dim=64, page_stride=4096, head_stride=1024, token_stride=64, dtype=L.BLK_BF16)
    return L.PagedCache(**(base | kw))


BAD_CACHES = [
    (dict(dtype=7), L.BLK_ERR_UNSUPPORTED), (dict(pages=-1), L.BLK_ERR_INVALID), (dict(pages=1 << 31), L.BLK_ERR_INVALID),
    (dict(page_size=0), L.BLK_ERR_INVALID), (dict(page_size=(1 << 30) + 1), L.BLK_ERR_INVALID), (dict(heads=0), L.BLK_ERR_INVALID),
    (dict(heads=1 << 16), L.BLK_ERR_INVALID), (dict(head_dim=0), L.BLK_ERR_UNSUPPORTED), (dict(head_dim=60), L.BLK_ERR_UNSUPPORTED),
    (dict(head_dim=6, dtype=L.BLK_F32), L.BLK_ERR_UNSUPPORTED), (dict(k=None), L.BLK_ERR_INVALID), (dict(v=None), L.BLK_ERR_INVALID),
    (dict(k=P + 8), L.BLK_ERR_UNALIGNED), (dict(page_stride=4097), L.BLK_ERR_UNALIGNED), (dict(head_stride=1028), L.BLK_ERR_UNALIGNED),
    (dict(token_stride=68), L.BLK_ERR_UNALIGNED), (dict(page_stride=-4096), L.BLK_ERR_INVALID)]


def attention(c, q=P, q_row=256, q_head=64, heads=4, table=P, stride=2, columns=2, lengths=P, requests=3, out=P, work=P, room=1 << 40):
    return L.lib.blk_paged_attention(C.byref(c) if c is not None else None, q, q_row, q_head, heads, table, stride, columns, lengths, requests, 1.0,
                                     out, None, work, room, None)


def append(c, k=P, k_row=256, k_head=64, v=P, v_row=256, v_head=64, slots=P, tokens=5):
    return L.lib.blk_paged_append(C.byref(c) if c is not None else None, k, k_row, k_head, v, v_row, v_head, slots, tokens, None)


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_caches(change, code):
    size = C.c_int64()
    assert attention(cache(**change)) == code
    assert append(cache(**change)) == code
    assert L.lib.blk_paged_attention_workspace(C.byref(cache(**change)), 4, 3, 2, C.byref(size)) == code
    assert L.lib.blk_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(heads=6), L.BLK_ERR_INVALID), (dict(heads=0), L.BLK_ERR_INVALID), (dict(heads=1 << 16), L.BLK_ERR_INVALID),
    (dict(requests=-1), L.BLK_ERR_INVALID), (dict(columns=-1), L.BLK_ERR_INVALID), (dict(columns=1 << 31), L.BLK_ERR_INVALID),
    (dict(q=None), L.BLK_ERR_INVALID), (dict(lengths=None), L.BLK_ERR_INVALID), (dict(out=None), L.BLK_ERR_INVALID),
    (dict(work=None), L.BLK_ERR_INVALID), (dict(table=None), L.BLK_ERR_INVALID), (dict(stride=-1), L.BLK_ERR_INVALID),
    (dict(q=P + 2), L.BLK_ERR_UNALIGNED), (dict(q_row=257), L.BLK_ERR_UNALIGNED), (dict(q_head=68), L.BLK_ERR_UNALIGNED),
    (dict(out=P + 8), L.BLK_ERR_UNALIGNED), (dict(work=P + 4), L.BLK_ERR_UNALIGNED)])
def test_attention(kw, code):
    assert attention(cache(), **kw) == code


def test_attention_heads_too_wide_and_nothing_to_do():
    assert attention(cache(head_dim=264, token_stride=264, head_stride=16 * 264, page_stride=64 * 264)) == L.BLK_ERR_UNSUPPORTED
    assert attention(None) == L.BLK_ERR_INVALID
    assert attention(cache(), requests=0) == L.BLK_OK


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), L.BLK_ERR_INVALID), (dict(tokens=1 << 31), L.BLK_ERR_INVALID), (dict(k=None), L.BLK_ERR_INVALID),
    (dict(v=None), L.BLK_ERR_INVALID), (dict(slots=None), L.BLK_ERR_INVALID), (dict(k=P + 2), L.BLK_ERR_UNALIGNED),
    (dict(v=P + 2), L.BLK_ERR_UNALIGNED), (dict(k_row=257), L.BLK_ERR_UNALIGNED), (dict(v_row=257), L.BLK_ERR_UNALIGNED),
    (dict(k_head=68), L.BLK_ERR_UNALIGNED), (dict(v_head=68), L.BLK_ERR_UNALIGNED)])
def test_append(kw, code):
    assert append(cache(), **kw) == code


@pytest.mark.parametrize("change", [dict(token_stride=56), dict(head_stride=1016), dict(page_stride=4088), dict(page_stride=0), dict(head_stride=0)])
def test_append_into_rows_that_overlap(change):
    assert append(cache(**change)) == L.BLK_ERR_INVALID
    assert b"overlap" in L.lib.blk_last_error()


def test_append_nothing():
    assert append(None) == L.BLK_ERR_INVALID
    assert append(cache(), tokens=0) == L.BLK_OK
    assert append(cache(pages=0, k=None, v=None)) == L.BLK_OK


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(columns=-1), dict(num_free=-1), dict(tokens=-1), dict(page_size=0), dict(page_size=(1 << 30) + 1), dict(table_stride=3),
    dict(lengths=None), dict(new=None), dict(table=None), dict(free=None), dict(taken=None), dict(slots=None), dict(lengths_out=None),
    dict(taken_out=None)])
def test_slots(kw):
    a = dict(lengths=P, new=P, requests=3, table=P, table_stride=4, columns=4, free=P, num_free=9, taken=P, page_size=16, slots=P, tokens=5,
             lengths_out=P, taken_out=P) | kw
    assert L.lib.blk_paged_slots(*a.values(), None) == L.BLK_ERR_INVALID


def test_host_tensors():
    f, i = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    c, t = torch.zeros(2, 4, 16, 64), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: blockPagedAttention(f, c, c, t, i), lambda: blockPagedAttention(f, c, c, t, i, return_lse=True),
                 lambda: blockPagedAppend(f, f, c, c, i.long()), lambda: blockPagedSlots(i, i, t, i, i[:1], 16, 2),
                 lambda: blockPagedAttention(f.numpy(), c, c, t, i), lambda: blockPagedSlots(np.zeros(2, np.int32), i, t, i, i[:1], 16, 2)):
        with pytest.raises(RuntimeError, match="must be CUDA Tensor"):
            call()


def test_attention_of_more_requests_than_its_indices_count():
    """The kernels count requests in 32 bits, up to a block's threads beyond the last one: as many as blk_paged_slots takes."""
    size = C.c_int64()
    for requests in ((1 << 31) - 1, (1 << 31) - 1024):
        assert attention(cache(), requests=requests) == L.BLK_ERR_INVALID
        assert L.lib.blk_paged_attention_workspace(C.byref(cache()), 4, requests, 2, C.byref(size)) == L.BLK_ERR_INVALID
        assert L.lib.blk_paged_slots(P, P, requests, P, 4, 4, P, 9, P, 16, P, 5, P, P, None) == L.BLK_ERR_INVALID
