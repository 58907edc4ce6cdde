"""GPU: the paged cache's attention where scores, weights or values are not ordinary numbers."""
import math

import pytest
import torch

from blockedattention_b200 import blockPagedAttention
from test_paged_gpu import BF16, F16, F32, check, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 4, 12])
@pytest.mark.parametrize("n", [3, 40, 700, 30000])
def test_logarithm_of_scores_of_minus_infinity(cuda_device, dtype, d, group, n):
    """ln sum exp of scores that are all -inf is -inf (the softmax is 0 / 0); a single other score is the logarithm then."""
    q, k, v, table, lengths = make([n] * 3 + [0], 1, group, d, 16, dtype)
    q[:] = 0.5
    k[table[:2, : -(-n // 16)].long()] = -math.inf
    k[table[1, (n - 1) // 16].long(), 0, (n - 1) % 16] = 0.0
    out, lse = blockPagedAttention(q, k, v, table, lengths, 0.125, return_lse=True)
    assert (lse[0] == -math.inf).all() and torch.isnan(out[0]).all()
    assert (lse[1] == 0).all() and torch.equal(out[1], v[table[1, (n - 1) // 16].long(), 0, (n - 1) % 16].expand(group, -1))
    assert torch.isfinite(lse[2]).all() and (lse[3] == -math.inf).all() and (out[3] == 0).all()
    k[table[0, 0].long(), 0, 1] = math.nan
    _, lse = blockPagedAttention(q, k, v, table, lengths, 0.125, return_lse=True)
    assert torch.isnan(lse[0]).all()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 64), (F16, 128), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("n", [16, 700, 30000])
@pytest.mark.parametrize("low", [-math.inf, -1000.0])
def test_tokens_without_weight_add_nothing(cuda_device, dtype, d, group, n, low):
    """One token of value zero among tokens whose weight is zero (a score of -inf, or e^-1000 of the largest, which no type here holds):
    zero exactly, however large their values and however many they are."""
    q, k, v, table, lengths = make([n], 1, group, d, 16, dtype)
    q[:] = 1.0
    k[:] = low / d
    v[:] = 60000.0
    page = table[0, n // 32].long()
    k[page, 0, 5] = 0.0
    v[page, 0, 5] = 0.0
    out, lse = blockPagedAttention(q, k, v, table, lengths, 1.0, return_lse=True)
    assert (out == 0).all() and (lse == 0).all()


@pytest.mark.parametrize("dtype,weight", [(F16, 2.0 ** -37), (BF16, 2.0 ** -100)])
def test_an_infinite_value_stays_one(cuda_device, dtype, weight):
    """Infinite values of tokens with small weights, also weights that the first of the two 16-bit numbers holds exactly."""
    for w in (weight, 2.0 ** -8, 0.7):
        q, k, v, table, lengths = make([700], 1, 2, 64, 16, dtype)
        q[:] = 0.0
        q[:, :, 0] = 1.0
        k[:] = 0.0
        v[:] = 1.0
        page = table[0, 20].long()
        k[page, 0, 5, 0] = math.log(w)
        v[page, 0, 5, 3], v[page, 0, 5, 4] = math.inf, -math.inf
        out = blockPagedAttention(q, k, v, table, lengths, 1.0)
        assert (out[..., 3] == math.inf).all() and (out[..., 4] == -math.inf).all()
        assert torch.isfinite(out[..., 5:]).all()


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("every", [False, True])
def test_weights_too_small_for_halves_are_rounded(cuda_device, group, every):
    """fp16: a weight is off by at most 2^-39 of the largest, in both directions: tokens of 2^-40.4 do not count as more than they may,
    be it behind one large score or with one in every tile, which all of them are relative to."""
    n = 30000
    q, k, v, table, lengths = make([n], 1, group, 64, 16, F16)
    q[:] = 1.0
    k[:] = -28.0 / 64
    v[:] = 60000.0
    large = table[0].long() if every else table[0, 900:901].long()
    k[large, 0, 5] = 0.0
    v[large, 0, 5] = 0.0
    out = blockPagedAttention(q, k, v, table, lengths, 1.0).double()
    small = (n - len(large)) / len(large)
    want = small * math.exp(-28.0) * 60000.0
    assert ((out - want).abs() <= (small + 1) * 2.0 ** -39 * 60000.0 + 2.0 ** -11 * want + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 4, 12])
@pytest.mark.parametrize("n", [3, 40, 700, 30000])
def test_logarithm_of_a_score_of_infinity(cuda_device, dtype, d, group, n):
    """ln sum exp with a score of +inf is +inf (the softmax is inf / inf: NaN), wherever the others stand, above or below zero; a NaN
    among them stays one."""
    q, k, v, table, lengths = make([n] * 4, 1, group, d, 16, dtype)
    q[:] = 8.0
    k[table[:, : -(-n // 16)].long()] = 3.0
    k[table[1].long()] = -3.0
    last = (table[:, (n - 1) // 16].long(), 0, (n - 1) % 16)
    k[last[0][:2], 0, last[2]] = math.inf
    k[table[2, 0].long(), 0, 0] = math.inf
    k[last[0][2], 0, last[2]] = -math.inf
    k[table[3, 0].long(), 0, 1] = math.inf
    k[table[3, 0].long(), 0, 2] = math.nan
    out, lse = blockPagedAttention(q, k, v, table, lengths, 1.0, return_lse=True)
    assert (lse[:3] == math.inf).all() and torch.isnan(lse[3]).all() and torch.isnan(out).all()


def windowed(window, lengths, kv, group, d, page, dtype, seed=0):
    """Long requests whose pages in front of the last ones are let go of, and what these hold on their own."""
    q, k, v, table, n = make(lengths, kv, group, d, page, dtype, seed)
    for r, x in enumerate(lengths):
        table[r, : max(0, x - window) // page] = -1
    held = [x - max(0, x - window) // page * page for x in lengths]
    only = torch.full((len(lengths), -(-max(held) // page)), -1, dtype=torch.int32, device="cuda")
    for r, (x, y) in enumerate(zip(lengths, held)):
        only[r, : -(-y // page)] = table[r, (x - y) // page: -(-x // page)]
    return q, k, v, table, n, only, ints(held)


@pytest.mark.parametrize("dtype,d,group", [(F16, 64, 1), (BF16, 128, 4), (BF16, 64, 24), (F32, 80, 2)])
@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("window", [1, 100, 4096])
def test_windows_that_begin_deep_in_long_requests(cuda_device, dtype, d, group, page, window):
    """Thousands of pages let go of: as the pages that are left give alone, to the tolerance of test_paged_gpu's check()."""
    q, k, v, table, n, only, held = windowed(window, [100000, 31, 57003, 0, 4096, 99991], 2, group, d, page, dtype)
    got = blockPagedAttention(q, k, v, table, n, d ** -0.5, return_lse=True)
    check(q, k, v, only, held, d ** -0.5, got)
    assert (got[0][3] == 0).all() and torch.equal(blockPagedAttention(q, k, v, table, n, d ** -0.5), got[0])


def test_logarithms_of_replays(cuda_device):
    """A captured call that gives logarithms, replayed with other queries, lengths and pages."""
    q, k, v, table, n = make([3000, 17, 0, 9000], 2, 4, 128, 16, BF16)
    blockPagedAttention(q, k, v, table, n, 0.09, return_lse=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = blockPagedAttention(q, k, v, table, n, 0.09, return_lse=True)
    for seed in range(3):
        now = make([[3000, 17, 0, 9000], [1, 8999, 64, 0], [65, 0, 2000, 4000]][seed], 2, 4, 128, 16, BF16, seed, columns=table.shape[1], spare=3)
        q.copy_(now[0])
        n.copy_(now[4])
        table.copy_(now[3].remainder(k.shape[0]))
        out.fill_(7), lse.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        check(q, k, v, table, n, 0.09, (out, lse))


def test_a_workspace_that_is_too_small(cuda_device):
    """The C entry refuses it on the host; with what it asks for, the call runs."""
    import ctypes as C

    from blockedattention_b200 import _lib as L
    q, k, v, table, n = make([300, 17], 2, 2, 64, 16, F16)
    want = blockPagedAttention(q, k, v, table, n, 0.125)
    cache = L.PagedCache(k.data_ptr(), v.data_ptr(), *(k.shape[i] for i in (0, 2, 1, 3)), k.stride(0), k.stride(1), k.stride(2), L.BLK_F16)
    size = C.c_int64()
    assert L.lib.blk_paged_attention_workspace(C.byref(cache), 4, 2, table.shape[1], C.byref(size)) == L.BLK_OK and size.value > 0
    work, out = torch.empty(size.value, dtype=torch.uint8, device="cuda"), torch.zeros_like(q)
    for room, code in ((size.value - 1, L.BLK_ERR_INVALID), (0, L.BLK_ERR_INVALID), (size.value, L.BLK_OK)):
        assert L.lib.blk_paged_attention(C.byref(cache), q.data_ptr(), q.stride(0), q.stride(1), 4, table.data_ptr(), table.stride(0), table.shape[1],
                                         n.data_ptr(), 2, 0.125, out.data_ptr(), None, work.data_ptr(), room,
                                         torch.cuda.current_stream().cuda_stream) == code
        torch.cuda.synchronize()
        assert torch.equal(out, want) if code == L.BLK_OK else (out == 0).all()


def test_threads_give_what_one_call_gives(cuda_device):
    """Calls from several threads on streams of their own: every one is compared, and an error in a thread is one here."""
    from concurrent.futures import ThreadPoolExecutor

    calls = [make([3000 + 100 * i, 17, 0], 2, 4, 64, 16, BF16, i) for i in range(4)]
    wants = [blockPagedAttention(*c, 0.125) for c in calls]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            return sum(torch.equal(blockPagedAttention(*calls[i], 0.125), wants[i]) for _ in range(30))

    with ThreadPoolExecutor(4) as pool:
        assert list(pool.map(work, range(4))) == [30] * 4


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F32, 64)])
@pytest.mark.parametrize("requests", [513, 5000, 40000])
def test_many_requests_of_a_few_tokens(cuda_device, dtype, d, requests):
    """Tens of thousands of requests of 0..4 tokens on one page each, by the definition in 64 bits."""
    g = torch.Generator("cuda").manual_seed(requests)
    k, v = (torch.randn((requests + 3, 2, 4, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((requests, 4, d), generator=g, device="cuda").to(dtype)
    table = torch.randperm(requests + 3, generator=g, device="cuda")[:requests].int()[:, None].contiguous()
    n = torch.randint(0, 5, (requests,), generator=g, device="cuda").int()
    out, lse = blockPagedAttention(q, k, v, table, n, d ** -0.5, return_lse=True)
    a, b = (c[table[:, 0].long()].double().repeat_interleave(2, 1) for c in (k, v))
    s = (a @ q.double()[..., None])[..., 0] * d ** -0.5
    s.masked_fill_(torch.arange(4, device="cuda") >= n[:, None, None], -math.inf)
    want = torch.nan_to_num(torch.softmax(s, -1))[:, :, None] @ b
    log = torch.logsumexp(s, -1)
    # (the tolerance of check(), with sums of at most 64 x 5 x 5 / 8 and values of at most 6)
    w = 2 * (d + 2) * 2.0 ** -23 * 200 + 2.0 ** -17 + 200 * 2.0 ** -23
    assert ((out.double() - want[:, :, 0]).abs() <= torch.finfo(dtype).eps / 2 * want[:, :, 0].abs() + 12 * w + 2.0 ** -25).all()
    some = (n > 0)[:, None].expand_as(lse)
    assert ((lse.double() - log)[some].abs() <= w + 2.0 ** -22 * 210).all() and (lse[~some] == -math.inf).all() and (out[n == 0] == 0).all()
