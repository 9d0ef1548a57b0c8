"""Paged cache on the GPU: append, attention over the cache, selected attention, against the
float64 forms of _paged_util (which also derives the bounds)."""

from __future__ import annotations

import math

import pytest
import torch

from tests._paged_util import ROUND, Case, assert_attention, rotate

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from dsa_b200 import device_status
    from dsa_b200.build import build

    build()
    device_status()
    yield
    assert device_status() == 0


def _attend(c, **kw):
    from dsa_b200.paged import paged_attention

    return paged_attention(c.qd, c.cache, c.batch, window=c.window, return_lse=True, **kw)


# ------------------------------------------------------------------ attention over the cache

@pytest.mark.parametrize("dtype,dim,hq,hkv,page", [
    (BF16, 128, 8, 2, 16), (F16, 64, 12, 4, 32), (BF16, 128, 5, 5, 64), (F16, 128, 40, 2, 128),
    (BF16, 64, 64, 1, 256), (BF16, 128, 64, 1, 1024)])
def test_one_token_per_sequence(dtype, dim, hq, hkv, page):
    c = Case([1, 1, 1, 1, 1, 1], [1, 15, 16, 17, 300, 1111], dtype=dtype, dim=dim, hq=hq,
             hkv=hkv, page=page)
    assert_attention(*_attend(c), c.reference(), dtype)


@pytest.mark.parametrize("dtype,dim,hq,hkv", [(BF16, 128, 16, 4), (F16, 64, 32, 4),
                                              (F16, 128, 32, 4), (BF16, 64, 4, 4)])
@pytest.mark.parametrize("batch", [3, 50])
@pytest.mark.parametrize("window", [None, 5, 70])
def test_a_few_tokens_per_sequence(dtype, dim, hq, hkv, batch, window):
    # up to 16 and up to 32 rows per key/value head, fewer and more items than SMs
    lens = [(37 * i) % 400 + 4 for i in range(batch)]
    c = Case([1 + i % 4 for i in range(batch)], lens, dtype=dtype, dim=dim, hq=hq, hkv=hkv,
             window=window, seed=16)
    assert_attention(*_attend(c), c.reference(), dtype)


@pytest.mark.parametrize("dtype,dim,hq,hkv,page", [
    (BF16, 128, 8, 2, 16), (F16, 64, 12, 4, 32), (BF16, 64, 7, 1, 16), (F16, 128, 10, 2, 64),
    (BF16, 128, 4, 4, 128), (BF16, 128, 132, 1, 256)])
@pytest.mark.parametrize("window", [None, 1, 37, 200])
def test_ragged_chunks(dtype, dim, hq, hkv, page, window):
    c = Case([3, 0, 1, 130, 64], [3, 20, 129, 257, 500], dtype=dtype, dim=dim, hq=hq, hkv=hkv,
             page=page, window=window, seed=3)
    assert_attention(*_attend(c), c.reference(), dtype)


@pytest.mark.parametrize("n", [2, 5, 17, 100])
def test_rows_without_keys_get_zeros(n):
    # more new tokens than positions: the first rows see nothing
    c = Case([n, 1, 2], [n // 2, 0, 1], seed=5)
    out, lse = _attend(c)
    assert_attention(out, lse, c.reference(), BF16)
    assert bool((out[:n - n // 2] == 0).all()) and bool((lse[:n - n // 2] == -math.inf).all())


def test_no_sequence_has_new_tokens():
    from dsa_b200.paged import paged_attention

    c = Case([0, 0], [7, 40])
    assert paged_attention(c.qd, c.cache, c.batch).shape == (0, 8, 128)


@pytest.mark.parametrize("max_new", [None, 1, 4, 70, 4096])
def test_result_does_not_depend_on_max_new(max_new):
    # the bound chooses a kernel; a wrong one must not change what is computed
    c = Case([70, 1, 4], [200, 333, 4], seed=8)
    c.batch.max_new = max_new
    assert_attention(*_attend(c), c.reference(), BF16)


@pytest.mark.parametrize("layout", ["hnd", "pair"])
@pytest.mark.parametrize("n", [1, 80])
def test_cache_layouts(layout, n):
    c = Case([n, 1], [150, 90], layout=layout, hkv=4, page=32, seed=2)
    assert not c.cache.keys.is_contiguous()
    assert_attention(*_attend(c), c.reference(), BF16)


@pytest.mark.parametrize("n", [1, 90])
def test_strided_queries_and_outputs(n):
    # q and out as slices of wider rows, heads not next to each other
    c = Case([n, 2], [200, 50], hq=6, hkv=2, seed=4)
    wide = torch.zeros(c.tokens, 7, 2, 128, dtype=BF16, device="cuda")
    wide[:, :6, 1] = c.qd
    room = torch.zeros(c.tokens, 9, 136, dtype=BF16, device="cuda")
    c.qd = wide[:, :6, 1]
    out, lse = _attend(c, out=room[:, 2:8, :128])
    assert_attention(out, lse, c.reference(), BF16)
    assert bool((room[:, :2] == 0).all()) and bool((room[:, 8:] == 0).all())
    assert bool((room[..., 128:] == 0).all())


@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_value_that_is_not_finite_reaches_only_the_tokens_that_see_it(n, value):
    # position 60 of 64 holds it; the tokens before it must not notice
    from dsa_b200.paged import paged_attention

    c = Case([n], [64], page=16, seed=6)
    clean = c.reference()
    slot = int(c.table[0, 60 // 16]), 60 % 16
    c.cache.values[slot[0], slot[1], 1, 5] = value
    out = paged_attention(c.qd, c.cache, c.batch)
    pos = torch.arange(64 - n, 64)
    sees = pos >= 60
    heads = torch.arange(8) >= 4
    hit = torch.zeros(n, 8, 128, dtype=torch.bool)
    hit[sees[:, None] & heads[None, :], 5] = True
    got = out.cpu()
    assert bool((~torch.isfinite(got[hit])).all())
    u = ROUND[BF16]
    err = (got.double() - clean[0]).abs()
    lim = (u + 2.0 ** -12) * clean[1] + u * (1 + u) * clean[0].abs() + 2.0 ** -24
    assert bool((err <= lim)[~hit].all())


def test_large_scores_do_not_overflow():
    c = Case([1, 33], [400, 120], seed=7)
    c.q = c.q * 30  # scores of hundreds: weights of all but a few keys vanish
    c.qd = c.q.cuda()
    out, lse = _attend(c)
    ref = c.reference()
    # the scores' rounding grows with them (|s| 2^-24 D): 30 x the bound of unit normals
    err = (out.double().cpu() - ref[0]).abs()
    u = ROUND[BF16]
    assert bool((err <= (u + 30 * 2.0 ** -12) * ref[1] + u * (1 + u) * ref[0].abs()).all())
    assert bool(((lse.double().cpu() - ref[2]).abs() <= 30 * 2.0 ** -12
                 + 2.0 ** -22 * ref[2].abs()).all())


@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_scale(scale):
    c = Case([1, 20], [100, 30], seed=9)
    out, lse = _attend(c, scale=scale)
    ref = c.reference(scale=scale)
    err = (out.double().cpu() - ref[0]).abs()
    u = ROUND[BF16]
    # scale 1: scores 11 times those of the default scale
    assert bool((err <= (u + 12 * 2.0 ** -12) * ref[1] + u * (1 + u) * ref[0].abs()).all())
    assert bool(((lse.double().cpu() - ref[2]).abs() <= 12 * 2.0 ** -12
                 + 2.0 ** -22 * ref[2].abs()).all())


def test_same_bits_every_time():
    c = Case([1] * 5 + [90], [900, 1, 3000, 77, 512, 1000], seed=10)
    first, lse = _attend(c)
    for _ in range(3):
        again, lse2 = _attend(c)
        assert torch.equal(first, again) and torch.equal(lse, lse2)


def test_other_streams_and_a_captured_graph():
    from dsa_b200.paged import paged_attention

    c = Case([1, 1], [500, 700], seed=11)
    want = c.reference()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = _attend(c)
    side.synchronize()
    assert_attention(out, lse, want, BF16)
    graph = torch.cuda.CUDAGraph()
    static = torch.empty_like(c.qd)
    with torch.cuda.graph(graph):
        paged_attention(c.qd, c.cache, c.batch, out=static)
    for lens in ([500, 700], [499, 3]):
        c.lens = lens
        c.batch.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        static.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert_attention(static, None, c.reference(), BF16)


def test_a_page_outside_the_cache_is_absent_and_reported():
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status

    for n in (1, 40):
        c = Case([n], [96], page=32, seed=12)
        c.batch.page_table[0, 1] = -1
        out, _ = _attend(c)
        assert device_status() & capi.TDSA_STATUS_RANGE
        idx = [[j for j in range(96 - n + i + 1) if not 32 <= j < 64] for i in range(n)]
        width = max(map(len, idx))
        ind = torch.tensor([r + [-1] * (width - len(r)) for r in idx])
        assert_attention(out, None, c.reference(indices=ind), BF16)


@pytest.mark.parametrize("n", [1, 2, 40])
def test_many_sequences(n):
    # more sequences than a block has threads, some with no new token or no position
    lens = [(7 * i) % 90 for i in range(900)]
    news = [0 if i % 5 == 2 else min(1 + i % n, max(lens[i], 1)) for i in range(900)]
    c = Case(news, lens, dim=64, hq=4, hkv=1, seed=14)
    assert_attention(*_attend(c), c.reference(), BF16)


@pytest.mark.parametrize("n", [1, 40])
def test_a_length_past_the_page_table_is_reported(n):
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status
    from dsa_b200.paged import PagedAppender

    c = Case([n, 1], [96, 20], page=32, seed=15)
    width = c.batch.page_table.shape[1] * 32
    for wrong in (width + 5, -3):
        c.batch.lengths[0] = wrong
        _attend(c)
        assert device_status() & capi.TDSA_STATUS_RANGE
        before = c.cache.keys.clone()
        k = torch.ones(n + 1, 2, 128, dtype=BF16, device="cuda")
        PagedAppender(c.cache, rope_dim=0).append(c.batch, k, k)
        assert device_status() & capi.TDSA_STATUS_RANGE
        changed = (c.cache.keys.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1)
        # the other sequence's token, and those of the first that the table still reaches
        slots = {(int(c.table[1, 19 // 32]), 19)}
        assert {tuple(x) for x in changed.nonzero().tolist()} <= slots | {
            (int(c.table[0, p // 32]), p % 32) for p in range(96)}
    c.batch.lengths[0] = 96
    device_status()


def test_offsets_past_32_bits():
    from dsa_b200.paged import PagedBatch, PagedKV, paged_attention

    pages = (1 << 31) // (64 * 2 * 128) + 70  # element offsets past 2^31
    store = torch.empty(2, pages, 64, 2, 128, dtype=BF16, device="cuda")
    c = Case([1, 100], [64, 130], page=64, seed=13)
    far = torch.full_like(c.batch.page_table, 0)
    n = 0
    for b, length in enumerate(c.lens):
        for i in range(-(-length // 64)):
            page = pages - 1 - n
            n += 1
            src = int(c.table[b, i])
            store[0, page], store[1, page] = c.cache.keys[src], c.cache.values[src]
            far[b, i] = page
    cache = PagedKV(store[0], store[1])
    batch = PagedBatch(far, c.batch.query_starts, c.batch.lengths, max_new=100)
    out, lse = paged_attention(c.qd, cache, batch, return_lse=True)
    assert_attention(out, lse, c.reference(), BF16)


# ------------------------------------------------------------------ selected attention

@pytest.mark.parametrize("dtype,dim,hq,hkv,page,index", [
    (BF16, 128, 8, 2, 16, torch.int32), (F16, 64, 12, 4, 32, torch.int64),
    (BF16, 64, 40, 1, 64, torch.int32), (F16, 128, 3, 3, 16, torch.int64)])
@pytest.mark.parametrize("k", [1, 16, 33, 257])
def test_selected_positions(dtype, dim, hq, hkv, page, index, k):
    from dsa_b200.paged import selected_attention

    c = Case([1, 7, 0, 2], [300, 65, 9, 2], dtype=dtype, dim=dim, hq=hq, hkv=hkv, page=page,
             seed=20 + k)
    g = torch.Generator().manual_seed(k)
    rows = []
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        for i in range(n):
            take = torch.randperm(length - n + i + 1, generator=g)[:k].sort().values
            rows.append(torch.nn.functional.pad(take, (0, k - take.numel()), value=-1))
    ind = torch.stack(rows)
    out, lse = selected_attention(c.qd, c.cache, c.batch, ind.to("cuda", index), return_lse=True)
    assert_attention(out, lse, c.reference(indices=ind), dtype)


@pytest.mark.parametrize("dtype,dim,hq,hkv", [(BF16, 128, 16, 8), (F16, 64, 16, 8),
                                              (F16, 128, 160, 8), (BF16, 64, 8, 8)])
@pytest.mark.parametrize("tokens", [30, 420])
@pytest.mark.parametrize("k", [22, 130])
def test_selected_positions_of_many_tokens(dtype, dim, hq, hkv, tokens, k):
    # an item per team of warps, split and whole, and an item per warp
    from dsa_b200.paged import selected_attention

    c = Case([tokens - 7, 0, 7], [tokens + 100, 3, 500], dtype=dtype, dim=dim, hq=hq, hkv=hkv,
             page=32, seed=21)
    g = torch.Generator().manual_seed(k)
    ind = torch.full((tokens, k), -1)
    for t in range(tokens):
        b = 0 if t < tokens - 7 else 2
        n = int(torch.randint(0, k + 1, (1,), generator=g))
        take = torch.randperm(c.lens[b], generator=g)[:n]
        ind[t, :take.numel()] = take
    out, lse = selected_attention(c.qd, c.cache, c.batch, ind.to("cuda", torch.int32),
                                  return_lse=True)
    assert_attention(out, lse, c.reference(indices=ind), dtype)


def test_selected_lists_in_any_order_with_gaps_and_repeats():
    from dsa_b200.paged import selected_attention

    c = Case([1, 1, 1], [200, 200, 50], seed=30)
    ind = torch.tensor([[199, -1, 3, 3, -5, 100, 0, 7], [-1] * 8, [49, 48, -1, 0, 0, 0, 1, 2]])
    wide = torch.full((3, 20), 77, dtype=torch.int32, device="cuda")
    wide[:, 4:12] = ind.cuda()
    out, lse = selected_attention(c.qd, c.cache, c.batch, wide[:, 4:12], return_lse=True)
    assert_attention(out, lse, c.reference(indices=ind), BF16)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


def test_selected_positions_past_the_length_are_skipped_and_reported():
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status
    from dsa_b200.paged import selected_attention

    c = Case([1, 1], [40, 20], seed=31)
    ind = torch.tensor([[0, 39, 40, 2 ** 40], [5, 20, 19, -1]])
    out, lse = selected_attention(c.qd, c.cache, c.batch, ind.cuda(), return_lse=True)
    assert device_status() & capi.TDSA_STATUS_RANGE
    assert_attention(out, lse, c.reference(indices=ind), BF16)


def test_rows_outside_every_sequence_are_left_alone():
    from dsa_b200.paged import paged_attention, selected_attention

    c = Case([2, 1], [30, 20], seed=32)
    q = torch.cat((torch.full_like(c.qd[:1], math.nan), c.qd, torch.full_like(c.qd[:2], math.nan)))
    c.batch.query_starts += 1
    ref = c.reference()
    for sel in (False, True):
        out = torch.full_like(q, 7.0)
        if sel:
            ind = torch.arange(30, dtype=torch.int32, device="cuda").repeat(6, 1)
            limit = torch.tensor([0, 28, 29, 19, 0, 0], device="cuda")[:, None]
            ind = torch.where(ind <= limit, ind, -1).to(torch.int32)
            selected_attention(q, c.cache, c.batch, ind, out=out)
        else:
            paged_attention(q, c.cache, c.batch, out=out)
        assert bool((out[[0, 4, 5]] == 7).all())
        assert_attention(out[1:4], None, ref, BF16)


def test_selection_of_every_position_equals_the_attention():
    from dsa_b200.paged import selected_attention

    c = Case([1, 1], [513, 77], seed=33)
    ind = torch.arange(513, dtype=torch.int32).repeat(2, 1)
    ind[1, 77:] = -1
    out, lse = selected_attention(c.qd, c.cache, c.batch, ind.cuda(), return_lse=True)
    assert_attention(out, lse, c.reference(), BF16)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("dtype,dim,hq,hkv,page", [
    (BF16, 128, 8, 2, 16), (F16, 64, 3, 3, 32), (BF16, 64, 20, 4, 64), (F16, 128, 1, 1, 128)])
@pytest.mark.parametrize("rope", [0, 16, 48, 64])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("news,lens", [([1, 0, 5, 40], [1, 3, 70, 41]),
                                       ([400, 0, 500], [450, 3, 600])])
def test_append(dtype, dim, hq, hkv, page, rope, interleaved, news, lens):
    from dsa_b200.paged import PagedAppender

    c = Case(news, lens, dtype=dtype, dim=dim, hq=hq, hkv=hkv, page=page, seed=40)
    g = torch.Generator().manual_seed(41)
    k = torch.randn(c.tokens, hkv, dim, generator=g).to(dtype)
    v = torch.randn(c.tokens, hkv, dim, generator=g).to(dtype)
    before = c.cache.keys.clone(), c.cache.values.clone()
    app = PagedAppender(c.cache, rope_dim=rope, interleaved=interleaved)
    q_out = app.append(c.batch, k.cuda(), v.cuda(), c.qd)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(c.news, c.lens)])
    freq = app.inv_freq.cpu()
    want_k, want_q = rotate(k, pos, freq, interleaved), rotate(c.q, pos, freq, interleaved)
    u = ROUND[dtype]

    def close(got, want, x):
        size = x.double().abs().amax(-1, keepdim=True)  # of any pair it is turned with
        err = (got.double().cpu() - want).abs()
        assert bool((err <= u * want.abs() + 2.0 ** -19 * size + 2.0 ** -25).all())

    close(q_out, want_q, c.q)
    seen = torch.zeros(before[0].shape[:2], dtype=torch.bool)
    t = 0
    for b, (n, m) in enumerate(zip(c.news, c.lens)):
        for p in range(m - n, m):
            at = int(c.table[b, p // page]), p % page
            seen[at] = True
            close(c.cache.keys[at][None], want_k[t][None], k[t][None])
            assert torch.equal(c.cache.values[at].cpu(), v[t])
            t += 1
    for now, was in zip((c.cache.keys, c.cache.values), before):  # nothing else was touched
        assert torch.equal(now[~seen.cuda()].view(torch.int16), was[~seen.cuda()].view(torch.int16))


def test_append_strides_positions_in_place_and_large_positions():
    from dsa_b200.paged import PagedAppender

    c = Case([3, 1], [10, 5], hq=4, hkv=2, layout="hnd", seed=42)
    qkv = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(1)).to(BF16)
    dev = qkv.cuda()
    pos = torch.tensor([131071, 1_000_003, 7, 0])
    app = PagedAppender(c.cache, rope_dim=128)
    ret = app.append(c.batch, dev[:, 4:6], dev[:, 6:], dev[:, :4], positions=pos.cuda(),
                     q_out=dev[:, :4])
    assert ret.data_ptr() == dev.data_ptr()
    want = rotate(qkv[:, :6], pos, app.inv_freq.cpu(), False)
    size = qkv[:, :6].double().abs().amax(-1, keepdim=True)
    err = (dev[:, :4].double().cpu() - want[:, :4]).abs()
    assert bool((err <= ROUND[BF16] * want[:, :4].abs() + 2.0 ** -19 * size[:, :4]).all())
    for t, (b, p) in enumerate([(0, 7), (0, 8), (0, 9), (1, 4)]):
        at = int(c.table[b, p // 16]), p % 16
        err = (c.cache.keys[at].double().cpu() - want[t, 4:6]).abs()
        assert bool((err <= ROUND[BF16] * want[t, 4:6].abs() + 2.0 ** -19 * size[t, 4:6]).all())
        assert torch.equal(c.cache.values[at].cpu(), qkv[t, 6:])


def test_append_reports_slots_that_are_not_there():
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status
    from dsa_b200.paged import PagedAppender

    c = Case([2, 1, 1], [1, 40, 40], seed=43)  # the first token has position -1
    c.batch.page_table[1, 39 // 16] = -1
    before = c.cache.keys.clone()
    k = torch.ones(4, 2, 128, dtype=BF16, device="cuda")
    PagedAppender(c.cache, rope_dim=0).append(c.batch, k, k)
    assert device_status() & capi.TDSA_STATUS_RANGE
    changed = (c.cache.keys.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1)
    want = torch.zeros_like(changed)
    want[int(c.table[0, 0]), 0] = True
    want[int(c.table[2, 39 // 16]), 39 % 16] = True
    assert torch.equal(changed, want)


# ------------------------------------------------------------------ refusals

def test_refusals():
    from dsa_b200.paged import (PagedAppender, PagedBatch, PagedKV, paged_attention,
                                selected_attention)

    c = Case([1, 1], [20, 30], seed=50)
    keys, values, q = c.cache.keys, c.cache.values, c.qd
    with pytest.raises(ValueError):
        PagedKV(keys, values.half())
    with pytest.raises(ValueError):
        PagedKV(keys.float(), values.float())
    with pytest.raises(ValueError):
        PagedKV(keys, values.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    with pytest.raises(ValueError):
        PagedKV(keys[0], values[0])
    with pytest.raises(ValueError):
        PagedBatch(c.batch.page_table.long(), c.batch.query_starts, c.batch.lengths)
    with pytest.raises(ValueError):
        PagedBatch(c.batch.page_table, c.batch.query_starts[:-1], c.batch.lengths)
    with pytest.raises(ValueError):
        PagedBatch(c.batch.page_table, c.batch.query_starts, c.batch.lengths, max_new=-1)
    for bad in (q.half(), q[..., :64], q[:, :7], q[0], q.cpu(), q.transpose(1, 2)):
        with pytest.raises(ValueError):
            paged_attention(bad, c.cache, c.batch)
    wide = torch.zeros(2, 8, 129, dtype=BF16, device="cuda")[..., 1:]
    with pytest.raises(ValueError):  # 16-byte alignment
        paged_attention(wide, c.cache, c.batch)
    with pytest.raises(ValueError):
        paged_attention(q, c.cache, c.batch, window=0)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            paged_attention(q, c.cache, c.batch, scale=scale)
    with pytest.raises(ValueError):
        paged_attention(q, c.cache, c.batch, out=torch.empty(3, 8, 128, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError):
        paged_attention(q, c.cache, c.batch, out=q)
    ind = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for bad in (ind[:1], ind.float(), ind[0], ind.cpu(), ind[:, :0], ind.t().contiguous().t()):
        with pytest.raises(ValueError):
            selected_attention(q, c.cache, c.batch, bad)
    with pytest.raises(ValueError):
        PagedAppender(c.cache, rope_dim=24)
    with pytest.raises(ValueError):
        PagedAppender(c.cache, rope_dim=256)
    with pytest.raises(ValueError):
        PagedAppender(c.cache, rope_dim=64, inv_freq=torch.ones(31, device="cuda"))
    app = PagedAppender(c.cache)
    k = torch.zeros(2, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        app.append(c.batch, k, k[:1])
    with pytest.raises(ValueError):
        app.append(c.batch, k, k, q_out=q)
    with pytest.raises(ValueError):
        app.append(c.batch, k, k, positions=torch.zeros(2, device="cuda"))
    # sizes this build does not have
    odd = torch.zeros(4, 24, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError):
        paged_attention(q, PagedKV(odd, odd.clone()), c.batch)
    odd = torch.zeros(4, 16, 2, 96, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError):
        paged_attention(torch.zeros(2, 8, 96, dtype=BF16, device="cuda"),
                        PagedKV(odd, odd.clone()), c.batch)
