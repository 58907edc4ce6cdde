"""GPU: the paged cache -- slots, writes and single-token attention -- against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from blockedattention_b200 import blockAttentionTokenMajor, blockPagedAppend, blockPagedAttention, blockPagedSlots

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I32 = torch.int32


def ints(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def make(lengths, kv, group, d, page, dtype, seed=0, layout="heads", columns=None, spare=3):
    """Caches with everything random, tables that name their pages in no order; -1 behind a request's last page."""
    g = torch.Generator("cuda").manual_seed(seed)
    held = [-(-max(n, 0) // page) for n in lengths]
    columns = max(held + [1]) if columns is None else columns
    order = np.random.RandomState(seed).permutation(sum(held) + spare)
    table, at = np.full((len(lengths), columns), -1), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n][:columns]
        at += n
    shape = (len(order), kv, page, d) if layout == "heads" else (len(order), page, kv, d)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if layout == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    q = torch.randn((len(lengths), kv * group, d), generator=g, device="cuda").to(dtype)
    return q, k, v, ints(table), ints(lengths)


def exact(q, k, v, table, lengths, scale):
    """(out, lse, S, V): the definition in 64 bits; sum |q k| |scale| and max |v| of each row, for the tolerance."""
    B, H, d = q.shape
    pages, kv, page, _ = k.shape
    out = torch.zeros((B, H, d), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    S, V = torch.zeros_like(lse), torch.zeros_like(lse)
    for r in range(B):
        n = min(max(int(lengths[r]), 0), table.shape[1] * page)
        place = torch.arange(n, device="cuda")
        named = table[r].long()[place // page] if n else place
        place, named = place[(named >= 0) & (named < pages)] % page, named[(named >= 0) & (named < pages)]
        if len(place) == 0:
            continue
        a = k[named, :, place].double().repeat_interleave(H // kv, 1).transpose(0, 1)  # (H, n, d)
        b = v[named, :, place].double().repeat_interleave(H // kv, 1).transpose(0, 1)
        x = q[r].double()[:, None] * a
        s = x.sum(-1) * scale
        out[r] = (torch.softmax(s, -1)[:, None] @ b)[:, 0]
        lse[r] = torch.logsumexp(s, -1)
        S[r] = x.abs().sum(-1).amax(-1) * abs(scale)
        V[r] = b.abs().amax((-1, -2))
    return out, lse, S, V


def check(q, k, v, table, lengths, scale, got=None):
    """A score is a sum of d products in 32 bits: off by at most (d + 2) 2^-23 of the sum of their sizes S (2^-23: a tensor core may cut
    where others round), as are its maximum's; the exponential and the 16-bit pair a weight enters as (2^-17), and the sums
    over the tokens, n / 16 terms in a row and some hundred parts, relative to themselves.  A relative error w of the weights moves the
    result by at most 2 w max |v|; it is rounded once, by half a unit."""
    out, lse = blockPagedAttention(q, k, v, table, lengths, scale, return_lse=True) if got is None else got
    want, log, S, V = exact(q, k, v, table, lengths, scale)
    n = int(lengths.max()) if lengths.numel() else 0
    w = 2 * (q.shape[2] + 2) * 2.0 ** -23 * S + 2.0 ** -17 + (n / 16 + 200) * 2.0 ** -23
    some = torch.isfinite(log)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == F32
    bound = torch.finfo(q.dtype).eps / 2 * want.abs() + (2 * w * V)[..., None] + (2.0 ** -25 if q.dtype == F16 else 0.0)  # (denormal halves)
    off = (out.double() - want).abs() - bound
    assert not torch.isnan(out).any() and off.max().item() <= 0, off.max().item()
    assert torch.equal(torch.isfinite(lse), some)
    assert (lse.double() - log)[some].abs().sub((w + 2.0 ** -22 * (S + log.abs()))[some]).max().item() <= 0 if some.any() else True
    assert (out[~some] == 0).all() and (lse[~some] == -math.inf).all()


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 100, 1000, 0, 2500, 31, 33, 128]


@pytest.mark.parametrize("dtype,d", [(t, d) for t in (F16, BF16) for d in (8, 40, 64, 72, 96, 128, 136, 192, 200, 256)] + [(F32, d) for d in (4, 20, 64, 100, 128, 200, 256)])
@pytest.mark.parametrize("kv,group,page,layout", [(1, 1, 16, "heads"), (3, 5, 24, "tokens"), (2, 8, 1, "heads"), (1, 17, 64, "tokens"), (2, 40, 100, "heads")])
def test_attention(cuda_device, dtype, d, kv, group, page, layout):
    check(*make(LENGTHS, kv, group, d, page, dtype, d + kv, layout), d ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 16, 23, 24, 25, 32, 33])
def test_groups_of_query_heads(cuda_device, dtype, group):
    check(*make([300, 1, 90], 2, group, 64, 16, dtype, group), 0.125)
    check(*make([300, 1, 90], 2, group, 128, 16, dtype, group), 0.09)
    check(*make([3000, 1, 90], 1, group, 256, 8, dtype, group), 0.06)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths", [[1], [64], [65], [20000], [150001, 3], [7] * 700, list(range(0, 1500)), [5000] * 40, [0] * 9, [0, 0, 40000, 0], [3, 0, 1, 2] * 1300])
@pytest.mark.parametrize("page", [16, 20])
def test_split_and_joined(cuda_device, dtype, lengths, page):
    check(*make(lengths, 2, 2, 64, page, dtype, len(lengths)), 0.125)


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 96), (BF16, 128), (F16, 192), (F16, 256), (F32, 64), (F32, 100), (F32, 256)])
@pytest.mark.parametrize("group", [1, 2, 4, 7, 12])
@pytest.mark.parametrize("page", [16, 6])
def test_heads_of_one_tile(cuda_device, dtype, d, group, page):
    """Batches in which nothing is longer than a tile, with and without one request that is; more and fewer of them than warps."""
    short = list(range(33)) * 3 if dtype == F32 and d > 64 else list(range(65)) * 3
    check(*make(short, 3, group, d, page, dtype, d), d ** -0.5)
    check(*make(short + [65], 3, group, d, page, dtype, d), d ** -0.5)
    check(*make([1, 0, 3], 1, group, d, page, dtype, d), d ** -0.5)


def test_no_requests(cuda_device):
    q, k, v, table, lengths = make([5], 1, 2, 64, 16, F16)
    out, lse = blockPagedAttention(q[:0], k, v, table[:0], lengths[:0], return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_pages_let_go_and_lengths_beyond_the_table(cuda_device, dtype):
    lengths = [200, 200, 200, 90, 64, 1 << 30, -5, 200, (1 << 31) - 1]
    q, k, v, table, _ = make([200] * 9, 2, 3, 64, 16, dtype)
    table[0, :5] = -1            # a window
    table[1, 3] = k.shape[0]     # no page of this cache
    table[2] = -1                # nothing left
    table[3, ::2] = -7
    table[4, :4] = -1            # all that it holds
    table[7, 1:12] = 1 << 30
    check(q, k, v, table, ints(lengths), 0.125)
    check(q, k, v, table[:, :0], ints(lengths), 0.125)   # a table without columns
    check(q, k[:0], v[:0], table, ints(lengths), 0.125)  # a cache without pages


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 72), (F32, 100)])
@pytest.mark.parametrize("page", [16, 24, 5])
def test_what_is_not_held_is_not_read(cuda_device, dtype, d, page):
    lengths = [0, 1, 17, 40, 63, 65, 300, 1]
    q, k, v, table, n = make(lengths, 2, 2, d, page, dtype)
    want = blockPagedAttention(q, k, v, table, n, 0.1)
    held = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for r, x in enumerate(lengths):
        for p in range(x):
            held[int(table[r, p // page]), p % page] = True
    for bad in (math.nan, math.inf, -math.inf):
        for c in (k, v):
            c.transpose(1, 2)[~held.cuda()] = bad
        assert torch.equal(blockPagedAttention(q, k, v, table, n, 0.1), want)


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0, 1e-30])
def test_scales(cuda_device, dtype, d, scale):
    check(*make([1, 70, 900], 2, 3, d, 16, dtype), scale)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_infinities_and_nan_stay_in_their_rows(cuda_device, dtype):
    q, k, v, table, n = make([300] * 6, 2, 4, 64, 16, dtype)
    want, log = blockPagedAttention(q, k, v, table, n, 0.125, return_lse=True)
    q[0, 1] = math.nan
    v[table[1, 2], 0, 3] = math.nan
    k[table[2, 2], 1, 3] = math.nan
    q[3] = 0.5
    k[table[3, :].long(), 0] = -math.inf          # every score -inf: 0 / 0
    k[table[4, 0].long(), 0] = 0
    q[4] = 0.5
    k[table[4, 0].long(), 0, 5, :] = -math.inf    # one token of -inf: no weight
    v[table[5, 1], 1, 2, 7] = math.inf
    out, lse = blockPagedAttention(q, k, v, table, n, 0.125, return_lse=True)
    assert torch.isnan(out[0, 1]).all() and torch.equal(out[0, [0, 2, 3, 4, 5, 6, 7]], want[0, [0, 2, 3, 4, 5, 6, 7]])
    assert torch.isnan(out[1, :4]).all() and torch.equal(out[1, 4:], want[1, 4:]) and torch.equal(lse[1], log[1])
    assert torch.isnan(out[2, 4:]).all() and torch.equal(out[2, :4], want[2, :4])
    assert torch.isnan(out[3, :4]).all() and torch.isfinite(out[3, 4:].float()).all()
    assert torch.isfinite(out[4].float()).all() and torch.isfinite(lse[4]).all()
    assert (out[5, 4:, 7] == math.inf).all() and torch.equal(out[5, 4:, :7], want[5, 4:, :7])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n", [40, 300, 30000])
def test_a_nan_is_not_lost_behind_large_scores(cuda_device, dtype, n):
    """A key of NaN among scores that have no weight (e^-1000 of the largest), in another warp, block or part than the largest; and keys of
    -inf alone there, which do have none."""
    q, k, v, table, lengths = make([n, n, n], 1, 2, 64, 16, dtype)
    q[:] = 1.0
    k[:] = 0.0
    k[table[:, 0].long(), 0, 0] = 16.0   # the first token's score: 1024
    k[table[0, n // 16 - 1], 0, 5] = math.nan
    k[table[1, 1:].long(), 0] = math.nan
    k[table[2, 1:].long(), 0] = -math.inf
    out, lse = blockPagedAttention(q, k, v, table, lengths, 1.0, return_lse=True)
    assert torch.isnan(out[:2]).all() and torch.isnan(lse[:2]).all()
    want = v[table[2, 0].long(), 0, 0].expand(2, -1)
    assert torch.equal(out[2], want) and (lse[2] == 1024).all()


def test_large_scores_and_one_token_over_many(cuda_device):
    # a page of large weights in front of many small ones, which halves hold only as multiples of 2^-24
    q, k, v, table, n = make([60000, 600], 1, 2, 64, 16, F16)
    q[:] = 1.0
    k[:] = 0.0
    k[table[0, 0].long(), 0, 0] = 0.25   # score 16 x 0.75 = 12: weight e^12 against 59999 of one
    v[:] = 1.0
    v[table[0, 0].long(), 0, 0] = -1.0
    check(q, k, v, table, n, 0.75)
    for dtype in (F16, BF16, F32):
        q, k, v, table, n = make([500, 90], 2, 2, 64, 16, dtype)
        check(q * 8, k, v, table, n, 1.0)


def test_views(cuda_device):
    B, kv, group, d, page = 5, 2, 4, 64, 16
    q, k, v, table, n = make([100, 3, 250, 64, 17], kv, group, d, page, BF16)
    want = blockPagedAttention(q, k, v, table, n, 0.125)
    fused = torch.randn((B, kv * (group + 2), d), device="cuda").to(BF16)   # queries, keys and values side by side
    fused[:, :kv * group] = q
    both = torch.stack([k, v], 1)                                           # (pages, 2, heads, page, d)
    wide = torch.full((B, table.shape[1] + 3), 1 << 20, dtype=I32, device="cuda")
    wide[:, 2:-1] = table
    assert torch.equal(blockPagedAttention(fused[:, :kv * group], both[:, 0], both[:, 1], wide[:, 2:-1], n, 0.125), want)
    backwards = both.flip(2)
    assert not torch.equal(blockPagedAttention(q, backwards[:, 0], backwards[:, 1], table, n, 0.125), want)
    same = q[:1].expand(B, -1, -1)                                          # one query for all
    assert torch.equal(blockPagedAttention(same, k, v, table, n, 0.125), blockPagedAttention(same.contiguous(), k, v, table, n, 0.125))
    one = table[:1].expand(3, -1)                                           # one document for all
    check(q[:3], k, v, one, ints([100, 50, 1]), 0.125)


def test_attention_offsets_beyond_32_bits(cuda_device):
    kv, d, page = 2, 64, 16
    step = (1 << 31) + (1 << 20)  # elements from page to page
    big = torch.empty(step + 2 * page * kv * d + 64, dtype=F16, device="cuda")
    k, v = (big[o:].as_strided((2, kv, page, d), (step, page * d, d, 1)) for o in (0, page * kv * d))
    g = torch.Generator("cuda").manual_seed(1)
    for c in (k, v):
        c.copy_(torch.randn((2, kv, page, d), generator=g, device="cuda"))
    q = torch.randn((2, 4, d), generator=g, device="cuda").half()
    check(q, k, v, ints([[0, 1], [1, 0]]), ints([32, 20]), 0.125)
    new = torch.randn((2, 3, kv, d), generator=g, device="cuda").half()
    before = k.clone()
    blockPagedAppend(new[0], new[1], k, v, torch.tensor([17, -1, 31], device="cuda"))
    before[1, :, 1], before[1, :, 15] = new[0, 0], new[0, 2]
    assert torch.equal(k, before) and torch.equal(v[1, :, 15], new[1, 2])


def test_slots_beyond_32_bits(cuda_device):
    # rows of 16 bytes: 2^31 + 64 of them are 34 GB
    rows = (1 << 31) + 64
    c = torch.empty((rows // 64, 1, 64, 8), dtype=F16, device="cuda")
    new = torch.randn((3, 1, 8), device="cuda").half()
    at = torch.tensor([rows - 1, 5, rows], device="cuda")
    blockPagedAppend(new, new, c, c, at)
    assert torch.equal(c[-1, 0, -1], new[0, 0]) and torch.equal(c[0, 0, 5], new[1, 0])
    slots, _, _ = blockPagedSlots(ints([100]), ints([2]), ints([[0, 0]]), ints([rows // 64 - 1]), ints([0]), 64, 2)
    assert slots.tolist() == [36, 37]
    slots, _, _ = blockPagedSlots(ints([63]), ints([3]), ints([[0, 0]]), ints([rows // 64 - 1]), ints([0]), 64, 3)
    assert slots.tolist() == [63, rows - 64, rows - 63]


def test_the_same_call_gives_the_same_bits_on_any_stream(cuda_device):
    q, k, v, table, n = make([3000, 17, 0, 9000], 2, 4, 128, 16, BF16)
    want = blockPagedAttention(q, k, v, table, n, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 4]):
            got.append(blockPagedAttention(q, k, v, table, n, 0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_two_graphs_replayed_at_once(cuda_device):
    calls = [make([3000, 17, 0, 9000], 2, 4, 128, 16, BF16, seed) for seed in (1, 2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    wants = [blockPagedAttention(*c, 0.09) for c in calls]
    torch.cuda.synchronize()
    for c, s in zip(calls, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(blockPagedAttention(*c, 0.09))
        graphs.append(graph)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    # lengths and pages are read when the graph runs
    q, k, v, table, n = calls[0]
    n.copy_(ints([8, 4000, 1, 0]))
    table.copy_(table.flip(0))
    graphs[0].replay()
    torch.cuda.synchronize()
    check(q, k, v, table, n, 0.09, (outs[0], blockPagedAttention(q, k, v, table, n, 0.09, return_lse=True)[1]))


def test_traced(cuda_device):
    """A trace records the attention as one node whose tensors are its inputs; what writes in place or gives two results is refused."""
    import warnings

    q, k, v, table, n = make([300, 17], 2, 2, 64, 16, F16)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(lambda *a: blockPagedAttention(*a, 0.125) * 2, (q, k, v, table, n))
        assert torch.equal(traced(q * 2, k, v, table, n - 5), blockPagedAttention(q * 2, k, v, table, n - 5, 0.125) * 2)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda q: blockPagedAttention(q, k, v, table, n, return_lse=True)[0], (q,))


def test_calls_from_several_threads(cuda_device):
    import threading

    calls = [make([3000 + 100 * i, 17, 0], 2, 4, 64, 16, BF16, i) for i in range(4)]
    wants = [blockPagedAttention(*c, 0.125) for c in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(blockPagedAttention(*calls[i], 0.125), wants[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ---- slots -----------------------------------------------------------------------------------------------
def plain_slots(lengths, new, table, free, taken, size, tokens):
    table, slots, out = np.array(table), [], []
    for r, (old, n) in enumerate(zip(lengths, new)):
        old, n = max(int(old), 0), max(int(n), 0)
        n = min(n, 2 ** 31 - 1 - old)
        for p in range(old, old + n):
            col = p // size
            if p % size == 0 and col < table.shape[1]:
                table[r, col] = max(free[taken], -1) if taken < len(free) else -1
                taken += 1
            page = table[r, col] if col < table.shape[1] else -1
            slots.append(int(page) * size + p % size if page >= 0 else -1)
        out.append(old + n)
    slots = (slots + [-1] * tokens)[:tokens]
    return slots, out, taken, table


def check_slots(lengths, new, columns, size, seed=0, tokens=None, free=None, taken=2, spare=5, advance=False):
    rs = np.random.RandomState(seed)
    lengths, new = np.asarray(lengths), np.asarray(new)
    table = rs.randint(0, 1000, (len(lengths), columns))
    for r, n in enumerate(lengths):
        table[r, min(columns, -(-max(int(n), 0) // size)):] = -9
    free = rs.permutation(int(sum(max(int(n), 0) // size + 1 for n in new)) + taken + spare) if free is None else np.asarray(free)
    tokens = int(np.maximum(new, 0).sum()) + 3 if tokens is None else tokens
    want = plain_slots(lengths, new, table, free, taken, size, tokens)
    args = [ints(lengths), ints(new), ints(table), ints(free), ints([taken])]
    versions = [t._version for t in args]
    slots, after, used = blockPagedSlots(*args, size, tokens, advance=advance)
    assert slots.dtype == torch.int64 and slots.tolist() == want[0]
    assert after.dtype == I32 and after.tolist() == want[1]
    assert used.tolist() == [want[2]]
    assert np.array_equal(args[2].cpu().numpy(), want[3])
    assert (after is args[0]) == advance and (used is args[4]) == advance
    if not advance:
        assert args[0].tolist() == list(lengths) and args[4].tolist() == [taken]
    assert [t._version > v for t, v in zip(args, versions)] == [advance, False, True, False, advance]


@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("size", [1, 3, 16, 100])
@pytest.mark.parametrize("requests,old,new", [(1, 0, 1), (1, 40, 1), (1, 5, 9000), (7, 100, 40), (64, 300, 1), (1024, 40, 2), (1025, 40, 2), (3000, 9, 30), (20, 0, 3000)])
def test_slots(cuda_device, requests, old, new, size, advance):
    rs = np.random.RandomState(requests + size)
    lengths, added = rs.randint(0, old + 1, requests), rs.randint(0, new + 1, requests)
    check_slots(lengths, added, -(-(old + new) // size), size, advance=advance)
    check_slots(lengths, np.ones_like(added), -(-(old + new) // size), size, advance=advance)


@pytest.mark.parametrize("advance", [False, True])
def test_slots_that_cannot_be(cuda_device, advance):
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 2, 16, advance=advance)                               # rows of the table full
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, free=[4, 8, 1], taken=1, advance=advance)      # pages used up
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, free=[], taken=0, advance=advance)
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, free=[4, -8, 1, -1, 3], taken=0, advance=advance)  # a list with holes
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, free=[4, 8, 1], taken=7, advance=advance)
    check_slots([-5, 0, 30, -7], [9, -40, 3, -1], 8, 16, advance=advance)                           # negative numbers are none
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, tokens=20, advance=advance)                    # fewer slots than tokens
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, tokens=0, advance=advance)
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 0, 16, advance=advance)                               # no columns
    check_slots([5, 0, 30, 7], [9, 40, 3, 1], 8, 16, tokens=50000, advance=advance)
    check_slots([0, 0], [20000, 20000], 3000, 16, tokens=9, advance=advance)
    check_slots([], [], 4, 16, tokens=5, advance=advance)
    check_slots([2 ** 31 - 3, 2 ** 31 - 1], [9, 0], 4, 1 << 30, advance=advance)                    # lengths end at 2^31 - 1


def test_slots_refuses(cuda_device):
    a = dict(lengths=ints([3, 4]), newTokens=ints([1, 1]), pageTable=ints([[0], [1]]), freePages=ints([2]), taken=ints([0]), pageSize=16, tokens=2)
    blockPagedSlots(**a)
    wide = ints(np.zeros((4, 4)))
    for bad in (dict(lengths=a["lengths"].long()), dict(lengths=ints([3])), dict(newTokens=ints([1, 1, 1])), dict(newTokens=wide[:2, 0]),
                dict(pageTable=ints([[0]])), dict(pageTable=wide.t()[:2, :2]), dict(pageTable=ints([0, 1])), dict(pageTable=wide[:1].expand(2, -1)),
                dict(pageTable=a["pageTable"].long()), dict(freePages=ints([[2]])), dict(taken=ints([0, 0])), dict(taken=ints([])),
                dict(pageSize=0), dict(pageSize=-1), dict(tokens=-1), dict(lengths=a["lengths"].cpu()), dict(freePages=a["freePages"].cpu())):
        with pytest.raises(RuntimeError):
            blockPagedSlots(**(a | bad))
    with pytest.raises(TypeError):
        blockPagedSlots(**(a | dict(tokens=2.5)))


# ---- append ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d", [(F16, 8), (BF16, 64), (F16, 72), (BF16, 128), (F32, 4), (F32, 72), (F32, 200), (F16, 520)])
@pytest.mark.parametrize("kv,page,tokens,layout", [(1, 16, 1, "heads"), (8, 16, 333, "tokens"), (3, 7, 100, "heads"), (2, 1, 50, "tokens"), (16, 64, 2000, "heads")])
def test_append(cuda_device, dtype, d, kv, page, tokens, layout):
    g = torch.Generator("cuda").manual_seed(tokens + d)
    pages = tokens // page + 3
    shape = (pages, kv, page, d) if layout == "heads" else (pages, page, kv, d)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if layout == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    fused = torch.randn((tokens, 3 * kv, d), generator=g, device="cuda").to(dtype)   # values, something else, keys
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[::7] = -1 - slots[::7]
    slots[3::11] += pages * page + (1 << 33)
    real = (slots >= 0) & (slots < pages * page)
    want = [k.clone(), v.clone()]
    for c, x in zip(want, (fused[:, 2 * kv:], fused[:, :kv])):
        c[slots[real] // page, :, slots[real] % page] = x[real]
    versions = k._version, v._version
    assert blockPagedAppend(fused[:, 2 * kv:], fused[:, :kv], k, v, slots) is None
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert k._version > versions[0] and v._version > versions[1]


def test_append_nothing(cuda_device):
    c = torch.zeros((2, 1, 16, 64), device="cuda")
    blockPagedAppend(c[0, :, :0].transpose(0, 1), c[0, :, :0].transpose(0, 1), c, c.clone(), torch.zeros(0, dtype=torch.int64, device="cuda"))
    blockPagedAppend(torch.ones((1, 1, 64), device="cuda"), torch.ones((1, 1, 64), device="cuda"), c[:0], c.clone()[:0], torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert (c == 0).all()


def test_append_refuses(cuda_device):
    k = torch.zeros((4, 2, 16, 64), dtype=F16, device="cuda")
    new, slots = torch.zeros((3, 2, 64), dtype=F16, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    a = dict(k=new, v=new, kCache=k, vCache=k.clone(), slots=slots)
    for bad in (dict(k=new[:2]), dict(k=new[:, :1]), dict(k=new[..., :32]), dict(k=new.float()), dict(v=new.bfloat16()), dict(k=new[0]),
                dict(k=new.transpose(1, 2).contiguous().transpose(1, 2)), dict(k=new.cpu()), dict(slots=slots.int()), dict(slots=slots[:2]),
                dict(slots=slots.cpu()), dict(kCache=k[:3]), dict(kCache=k.float()), dict(kCache=k.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(kCache=k[0]), dict(kCache=k.cpu()), dict(kCache=k[:1].expand(4, -1, -1, -1), vCache=k[:1].expand(4, -1, -1, -1)),
                dict(kCache=torch.zeros_like(k, requires_grad=True)), dict(kCache=k.int(), vCache=k.int(), k=new.int(), v=new.int())):
        with pytest.raises(RuntimeError):
            blockPagedAppend(**(a | bad))
    odd = torch.zeros(k.numel() + 4, dtype=F16, device="cuda")[4:].view(k.shape)
    with pytest.raises(RuntimeError, match="16-byte"):
        blockPagedAppend(**(a | dict(kCache=odd, vCache=odd.clone())))


def test_attention_refuses(cuda_device):
    q, k, v, table, n = make([30, 40], 2, 2, 64, 16, F16)
    a = dict(q=q, kCache=k, vCache=v, pageTable=table, lengths=n)
    odd = torch.zeros(q.numel() + 4, dtype=F16, device="cuda")[4:].view(q.shape)
    for bad in (dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.bfloat16()), dict(q=q.cpu()), dict(q=odd), dict(q=q[0]), dict(q=q[:, :0]),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(kCache=k[:, :1]), dict(vCache=v.float()), dict(vCache=v[:-1]),
                dict(vCache=v.transpose(1, 2).contiguous().transpose(1, 2)), dict(kCache=k[..., ::2], vCache=v[..., ::2], q=q[..., :32]),
                dict(pageTable=table[:1]), dict(pageTable=table.long()), dict(pageTable=table[0]), dict(pageTable=table.repeat(1, 2)[:, ::2]),
                dict(pageTable=table.cpu()), dict(lengths=n[:1]), dict(lengths=n.long()), dict(lengths=ints([3, 4, 5, 6])[::2]),
                dict(kCache=k.double(), vCache=v.double(), q=q.double())):
        for lse in (False, True):
            with pytest.raises(RuntimeError):
                blockPagedAttention(**(a | bad), return_lse=lse)
    with pytest.raises(RuntimeError, match="256"):
        blockPagedAttention(torch.zeros((2, 2, 264), device="cuda"), torch.zeros((4, 1, 16, 264), device="cuda"), torch.zeros((4, 1, 16, 264), device="cuda"), table, n)


# ---- together --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,layout", [(F16, "heads"), (BF16, "tokens")])
def test_prompts_then_steps(cuda_device, dtype, layout):
    """Packed prompts through the framework's attention, their keys and values kept, then steps of one token: the first ones call
    by call, the others as replays of one captured step."""
    H, group, d, page, steps = 2, 2, 64, 16, 20
    prompts = np.array([1, 50, 16, 33, 7])
    B, total = len(prompts), int(prompts.sum())
    g = torch.Generator("cuda").manual_seed(4)
    x = [torch.randn((total, H, d), generator=g, device="cuda").to(dtype) for _ in range(3)]
    encoded = blockAttentionTokenMajor(*x, prompts, scale=d ** -0.5)
    assert torch.isfinite(encoded).all()
    pages = 30
    shape = (pages, H, page, d) if layout == "heads" else (pages, page, H, d)
    k, v = (torch.full(shape, math.nan, device="cuda", dtype=dtype) for _ in range(2))
    if layout == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    lengths, taken = ints([0] * B), ints([0])
    table, free = ints(np.full((B, 6), -1)), torch.randperm(pages, generator=g, device="cuda").int()
    slots, _, _ = blockPagedSlots(lengths, ints(prompts), table, free, taken, page, total, advance=True)
    blockPagedAppend(x[1], x[2], k, v, slots)
    history = [[list(t) for t in zip(*(c.split(prompts.tolist())[r] for c in (x[1], x[2])))] for r in range(B)]
    one = ints([1] * B)
    new = [torch.zeros((B, n, d), dtype=dtype, device="cuda") for n in (H * group, H, H)]

    def step():
        slots, now, _ = blockPagedSlots(lengths, one, table, free, taken, page, B, advance=True)
        blockPagedAppend(new[1], new[2], k, v, slots)
        return blockPagedAttention(new[0], k, v, table, now, d ** -0.5)

    graph = None
    for i in range(steps):
        for t in new:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        if i < 3:
            out = step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step()
            graph.replay()
        for r in range(B):
            history[r].append([new[1][r].clone(), new[2][r].clone()])
            a, b = (torch.stack([t[j] for t in history[r]]).double().repeat_interleave(group, 1).transpose(0, 1) for j in range(2))
            want = (torch.softmax((new[0][r].double()[:, None] * a).sum(-1) * d ** -0.5, -1)[:, None] @ b)[:, 0]
            # (the tolerance of check(), with sums of at most 40 and values of at most 5)
            assert ((out[r].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 10 * (132 * 2.0 ** -23 * 40 + 2.0 ** -17 + 2.0 ** -15)).all()
    assert lengths.tolist() == [int(p) + steps for p in prompts]
    assert taken.tolist() == [sum(-(-(int(p) + steps) // page) for p in prompts)]
    assert len({int(p) for p in table.flatten().tolist() if p >= 0}) == int(taken)


def test_lists_remembered_from_a_tensor_that_is_advanced(cuda_device):
    """A list read from a GPU tensor is remembered under its version: after a step in place its new values count."""
    lengths, taken = ints([3, 5]), ints([0])
    table = ints(np.full((2, 2), -1))
    q = torch.randn((10, 2, 64), device="cuda").half()
    a = blockAttentionTokenMajor(q[:8], q[:8], q[:8], lengths, scale=0.125)
    blockPagedSlots(lengths, ints([1, 1]), table, ints([0, 1]), taken, 16, 2, advance=True)
    b = blockAttentionTokenMajor(q, q, q, lengths, scale=0.125)
    assert a.shape[0] == 8 and torch.equal(b, blockAttentionTokenMajor(q, q, q, [4, 6], scale=0.125))
