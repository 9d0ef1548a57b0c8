"""Paged cache on the GPU where it can go wrong: keys, queries and values that are not finite or
huge, weights far below a row's largest, windows and lengths at the ends of their ranges, long
chunks.  Against the float64 forms of _paged_util, whose bounds hold unless a test says more."""

from __future__ import annotations

import math

import pytest
import torch

from tests._paged_util import ROUND, Case, rotate

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


def _set(c, which, b, pos, head, feature, value):
    """One number of the cache, in its pages and in the float64 copy."""
    store, copy = (c.cache.keys, c.k) if which == "k" else (c.cache.values, c.v)
    store[int(c.table[b, pos // c.page]), pos % c.page, head, feature] = value
    copy[b][pos, head, feature] = value


def _check(c, got, want, extra=0.0):
    """Like assert_attention, where the reference's sums may be NaN or infinite: NaN has to be
    NaN, infinity the same infinity, a log-sum-exp that is not finite any such number.  extra:
    more room for the outputs."""
    (out, lse), (ref, mag, ref_lse) = got, want
    out, u = out.double().cpu(), ROUND[c.dtype]
    lim = (u + 2.0 ** -12) * mag + u * (1 + u) * ref.abs() + 2.0 ** -24 + extra
    fine = torch.isfinite(ref)
    assert bool(((out - ref).abs() <= lim)[fine].all())
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(out[torch.isinf(ref)], ref[torch.isinf(ref)])
    lse = lse.double().cpu()
    empty, odd = ref_lse == -math.inf, torch.isnan(ref_lse) | (ref_lse == math.inf)
    assert torch.equal(lse == -math.inf, empty)
    assert not torch.isfinite(lse[odd]).any()
    e = (lse - ref_lse)[~empty & ~odd].abs()
    assert bool((e <= 2.0 ** -12 + 2.0 ** -22 * ref_lse[~empty & ~odd].abs()).all())


# ------------------------------------------------------------------ scores that are not finite

@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n", [1, 8, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_key_that_is_not_finite_reaches_the_rows_that_see_it(dtype, dim, n, value):
    # at each of 32 consecutive positions, the last of which only some of the tokens see: a NaN
    # or +inf score makes its row NaN, a score of -inf weighs nothing
    c = Case([n, 2], [160, 30], dtype=dtype, dim=dim, seed=60)
    for pos in range(160 - 16 - 32, 160 - 16) if n > 16 else range(100, 132):
        was = float(c.k[0][pos, 1, 3])
        _set(c, "k", 0, pos, 1, 3, value)
        _check(c, _attend(c), c.reference())
        _set(c, "k", 0, pos, 1, 3, was)


@pytest.mark.parametrize("n", [1, 40])
def test_a_key_that_is_not_finite_outside_the_window(n):
    c = Case([n], [300], seed=61, window=33)
    for pos in (5, 255, 259, 262, 264, 266, 280, 299):
        was = float(c.k[0][pos, 0, 7])
        _set(c, "k", 0, pos, 0, 7, math.nan)
        _check(c, _attend(c), c.reference())
        _set(c, "k", 0, pos, 0, 7, was)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_query_that_is_not_finite_stays_in_its_row(n, value):
    c = Case([n, n], [200, 77], dtype=F16, seed=62)
    c.q[n // 2, 3, 9] = value
    c.qd = c.q.cuda()
    _check(c, _attend(c), c.reference())


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_key_that_is_not_finite_in_a_split_sequence(value):
    # many parts of one item, one of which holds it
    c = Case([40], [3000], dim=64, hq=4, hkv=1, seed=63)
    for pos in (2, 1025, 2990):
        was = float(c.k[0][pos, 0, 0])
        _set(c, "k", 0, pos, 0, 0, value)
        _check(c, _attend(c), c.reference())
        _set(c, "k", 0, pos, 0, 0, was)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_keys_that_are_not_finite_in_whole_items(dtype, value):
    # items of one unit each, of which none is split: sequence b has it at position 50 + b
    c = Case([40] * 36, [100] * 36, dtype=dtype, dim=64, hq=16, hkv=8, seed=75)
    for b in range(36):
        _set(c, "k", b, 50 + b, b % 8, 3, value)
    _check(c, _attend(c), c.reference())


# ------------------------------------------------------------------ weights of nothing

@pytest.mark.parametrize("n", [8, 40])
def test_a_huge_value_reaches_only_the_tokens_that_see_it(n):
    # the largest bfloat16 at each of the last positions: nothing of it in earlier tokens
    c = Case([n], [160], seed=64)
    clean = c.reference()
    for pos in range(160 - min(n, 32), 160):
        was = float(c.v[0][pos, 1, 5])
        _set(c, "v", 0, pos, 1, 5, torch.finfo(BF16).max)
        out, lse = _attend(c)
        hidden = torch.arange(160 - n, 160) < pos
        _check(c, (out[hidden.cuda()], lse[hidden.cuda()]), tuple(x[hidden] for x in clean))
        _set(c, "v", 0, pos, 1, 5, was)


@pytest.mark.parametrize("n", [1, 40])
def test_a_weight_below_the_type_times_a_huge_value(n):
    # scores 283 below the others': a weight of 2^-408 times the largest bfloat16 is nothing
    c = Case([n], [200], dim=128, hq=2, hkv=1, seed=65)
    c.q[..., 0] = 8.0
    c.qd = c.q.cuda()
    for pos in range(64, 96):
        was = float(c.k[0][pos, 0, 0]), float(c.v[0][pos, 0, 2])
        _set(c, "k", 0, pos, 0, 0, -400.0)
        _set(c, "v", 0, pos, 0, 2, torch.finfo(BF16).max)
        # the other scores' first products are up to 8 times a unit normal's
        ref = c.reference()
        _check(c, _attend(c), ref, extra=2.0 ** -9 * ref[1])
        _set(c, "k", 0, pos, 0, 0, was[0])
        _set(c, "v", 0, pos, 0, 2, was[1])


# ------------------------------------------------------------------ a long tail of small weights

def _sink(n, length, dtype, dim, gap, tail=0.0):
    """One key ``gap`` above all the others with a value of zero, and values of 1 behind it."""
    c = Case([n], [length], dtype=dtype, dim=dim, hq=4, hkv=1, page=64, seed=66)
    c.q[..., 0], c.q[..., 1:] = math.sqrt(dim), c.q[..., 1:] * tail
    c.qd = c.q.cuda()
    keys, values = c.k[0], c.v[0]
    keys[:, :, 0], keys[0, :, 0] = 0.0, gap
    keys[:, :, 1:] *= tail
    keys.copy_(keys.to(dtype).double())
    values[:], values[0] = 1.0, 0.0
    pages = c.table[0, :-(-length // 64)].long().cuda()
    for store, rows in ((c.cache.keys, keys), (c.cache.values, values)):
        room = torch.zeros(pages.numel() * 64, 1, dim, dtype=dtype)
        room[:length] = rows.to(dtype)
        store[pages] = room.view(-1, 64, 1, dim).cuda()
    return c


# 16-bit weights hold 2^-11 (or 2^-8) of themselves down to 2^-25 of the row's largest, and below
# that, in float16, half of its smallest number, which stands for 2^-36 of the row's largest
def _tail_room(c):
    return 2.0 ** -36 * c.lens[0]


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("gap", [8.0, 13.9, 17.40625])
def test_a_long_tail_of_small_weights_is_kept(dtype, dim, n, gap):
    c = _sink(n, 20000 if n < 40 else 6000, dtype, dim, gap)
    _check(c, _attend(c), c.reference(), extra=_tail_room(c))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 40])
def test_a_tail_of_many_weights_is_kept(dtype, n):
    # scores that spread, so that a row's largest grows along the way
    c = _sink(n, 6000, dtype, 64, 14.0, tail=0.6)
    _check(c, _attend(c), c.reference(), extra=_tail_room(c))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_tail_of_selected_positions_is_kept(dtype):
    from dsa_b200.paged import selected_attention

    c = _sink(5, 4000, dtype, 64, 15.0)
    ind = torch.stack([torch.randperm(4000, generator=torch.Generator().manual_seed(i))
                       for i in range(5)])
    got = selected_attention(c.qd, c.cache, c.batch, ind.cuda(), return_lse=True)
    _check(c, got, c.reference(indices=ind), extra=_tail_room(c))


@pytest.mark.parametrize("n", [1, 8, 40])
def test_a_value_near_the_types_largest_does_not_overflow(n):
    # half of a row's weight on the largest bfloat16: products with weights above 1 would be
    # infinite
    c = Case([n], [160], dim=64, hq=4, hkv=1, seed=76)
    c.q[..., 0] = 8.0
    c.qd = c.q.cuda()
    for pos in (40, 50, 66, 83, 101, 118):
        was = float(c.k[0][pos, 0, 0]), float(c.v[0][pos, 0, 2])
        _set(c, "k", 0, pos, 0, 0, 5.0)
        _set(c, "v", 0, pos, 0, 2, torch.finfo(BF16).max)
        ref = c.reference()
        _check(c, _attend(c), ref, extra=2.0 ** -9 * ref[1])  # scores 8 times a unit normal's
        _set(c, "k", 0, pos, 0, 0, was[0])
        _set(c, "v", 0, pos, 0, 2, was[1])


# ------------------------------------------------------------------ after a wait that ran out

@pytest.mark.parametrize("n", [1, 40])
def test_calls_after_a_timeout_do_not_find_its_counters(monkeypatch, n):
    # arrival counters as a call that ended early may leave them, and the status that reports it
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status, paged

    c = Case([n], [3000], dim=64, hq=4, hkv=1, seed=77)
    _check(c, _attend(c), c.reference())
    for buffer, _, _ in paged._WORKSPACES.values():
        buffer[:capi.TDSA_PAGED_COUNTER_BYTES].view(torch.int32).fill_(999)
    with monkeypatch.context() as m:
        m.setattr(capi, "device_status", lambda reset=True: capi.TDSA_ERR_TIMEOUT)
        assert device_status() == capi.TDSA_ERR_TIMEOUT
    try:
        _check(c, _attend(c, out=torch.full_like(c.qd, math.nan)), c.reference())
    finally:
        paged._WORKSPACES.clear()


# ------------------------------------------------------------------ ends of ranges

@pytest.mark.parametrize("news,lens", [([1, 3], [300, 1]), ([40, 9], [300, 4])])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 32,
                                    2 ** 32 + 5, 2 ** 70])
def test_a_window_past_every_position_is_none(news, lens, window):
    # the second sequence has more new tokens than positions
    c = Case(news, lens, seed=67)
    c.window = window
    got = _attend(c)
    c.window = None
    _check(c, got, c.reference())


@pytest.mark.parametrize("n", [2, 9])
def test_a_window_of_the_c_ints_range(n):
    # the C entry's own range ends at 2^31 - 1
    import ctypes as C

    from dsa_b200 import _capi as capi
    from dsa_b200.indexer import stream_ptr
    from dsa_b200.paged import paged_workspace

    c = Case([n], [1], seed=78)
    out, lse = torch.zeros_like(c.qd), torch.zeros(n, 8, device="cuda")
    rows = [capi.TdsaTokenRows(t.data_ptr(), *t.stride()[:2]) for t in (c.qd, out)]
    ws = paged_workspace(c.cache.device, 128)
    rc = capi.lib().tdsa_paged_attention(
        c.cache._ref, c.batch._for(n), C.byref(rows[0]), 8, 128 ** -0.5, 2 ** 31 - 1,
        C.byref(rows[1]), lse.data_ptr(), ws[1], ws[2], stream_ptr(c.cache.device))
    assert rc == 0
    _check(c, (out, lse), c.reference())


@pytest.mark.parametrize("n", [1, 7, 40])
@pytest.mark.parametrize("window", [None, 38])
@pytest.mark.parametrize("past", [1, 5, 2 ** 31 - 1 - 128])
def test_a_length_past_the_page_table_keeps_the_tokens_positions(n, window, past):
    # positions from the table's end on are absent; the tokens stay where the length puts them
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status

    c = Case([n, 2], [96, 30], page=32, window=window, seed=68)
    length = 128 + past  # the table reaches 128, of which the last page is not one of the cache's
    c.batch.lengths[0] = length
    got = _attend(c)
    assert device_status() & capi.TDSA_STATUS_RANGE
    rows = []
    for b, (new, end) in enumerate(((n, length), (2, 30))):
        for i in range(new):
            pos = end - new + i
            lo = 0 if window is None else max(0, pos - window + 1)
            rows.append(list(range(min(lo, 96), min(pos + 1, 96))))
    width = max(map(len, rows))
    ind = torch.tensor([r + [-1] * (width - len(r)) for r in rows]).view(len(rows), width)
    _check(c, got, c.reference(indices=ind))


def test_append_turns_queries_by_positions_before_the_first():
    # more new tokens than positions: no slot for the first ones, but a position all the same
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status
    from dsa_b200.paged import PagedAppender

    c = Case([9, 1], [4, 20], hq=4, hkv=2, seed=69)
    k = torch.randn(10, 2, 128, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    app = PagedAppender(c.cache, rope_dim=128)
    got = app.append(c.batch, k, k, c.qd)
    assert device_status() & capi.TDSA_STATUS_RANGE
    pos = torch.cat((torch.arange(-5, 4), torch.tensor([19])))
    want = rotate(c.q, pos, app.inv_freq.cpu(), False)
    size = c.q.double().abs().amax(-1, keepdim=True)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= ROUND[BF16] * want.abs() + 2.0 ** -19 * size + 2.0 ** -25).all())


# ------------------------------------------------------------------ outputs beside their inputs

@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("way", ["heads", "features", "tokens", "head-major"])
def test_outputs_in_the_same_buffer_as_queries(n, way):
    # interleaved in every way, and nowhere the same memory
    c = Case([n, 2], [90, 30], hq=8, hkv=2, seed=79)
    t = c.tokens
    if way == "heads":
        room = torch.zeros(t, 16, 128, dtype=BF16, device="cuda")
        q, out = room[:, :8], room[:, 8:]
    elif way == "features":
        room = torch.zeros(t, 8, 2, 128, dtype=BF16, device="cuda")
        q, out = room[:, :, 0], room[:, :, 1]
    elif way == "tokens":
        room = torch.zeros(t, 2, 8, 128, dtype=BF16, device="cuda")
        q, out = room[:, 1], room[:, 0]
    else:
        room = torch.zeros(8, 2, t, 128, dtype=BF16, device="cuda")
        q, out = room[:, 0].transpose(0, 1), room[:, 1].transpose(0, 1)
    q.copy_(c.qd)
    c.qd = q
    _check(c, _attend(c, out=out), c.reference())
    assert torch.equal(q.cpu(), c.q)


# ------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F16, 128)])
@pytest.mark.parametrize("n", [1, 8, 40])
def test_an_infinite_value_is_infinite_where_it_is_seen(dtype, dim, n):
    # +inf in one feature, -inf in another, both in a third: inf, -inf and NaN
    c = Case([n, 3], [170, 40], dtype=dtype, dim=dim, seed=70)
    for pos in (0, 17, 100, 135, 150, 160, 169):
        _set(c, "v", 0, pos, 1, 5, math.inf)
    for pos in (150, 168):
        _set(c, "v", 0, pos, 1, 6, math.inf)
    for pos in (3, 120, 140, 165):
        _set(c, "v", 0, pos, 1, 9, -math.inf)
    _set(c, "v", 0, 20, 0, 30, math.inf)
    _set(c, "v", 0, 151, 0, 30, -math.inf)
    _set(c, "v", 0, 155, 0, 31, math.nan)
    _check(c, _attend(c), c.reference())


@pytest.mark.parametrize("tokens", [3, 400])
def test_an_infinite_value_among_selected_positions(tokens):
    from dsa_b200.paged import selected_attention

    c = Case([tokens], [450], hq=16, hkv=8, dim=64, seed=71)
    for head in range(8):
        _set(c, "v", 0, 7 * head + 30, head, 5, math.inf)
        _set(c, "v", 0, 7 * head + 31, head, 5 + head, -math.inf)
    g = torch.Generator().manual_seed(72)
    ind = torch.stack([torch.randperm(450, generator=g)[:60] for _ in range(tokens)])
    got = selected_attention(c.qd, c.cache, c.batch, ind.cuda(), return_lse=True)
    _check(c, got, c.reference(indices=ind))


# ------------------------------------------------------------------ long chunks

def _torch_reference(c):
    """Case.reference a head at a time for all tokens of a sequence, on the GPU in float64."""
    g = c.hq // c.hkv
    out = torch.zeros(c.tokens, c.hq, c.dim, dtype=torch.float64)
    mag, lse = torch.zeros_like(out), torch.full((c.tokens, c.hq), -math.inf, dtype=torch.float64)
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")
        sees = (j <= pos) & c.there[b].cuda()
        if c.window is not None:
            sees &= j > pos - c.window
        rows = slice(c.starts[b], c.starts[b] + n)
        for h in range(c.hq):
            k, v = c.k[b][:, h // g].cuda(), c.v[b][:, h // g].cuda()
            z = (c.q[rows, h].double().cuda() @ k.T * c.dim ** -0.5).masked_fill(~sees, -math.inf)
            w = torch.softmax(z, -1).nan_to_num(0.0)
            out[rows, h], mag[rows, h] = (w @ v).cpu(), (w @ v.abs()).cpu()
            lse[rows, h] = torch.logsumexp(z, -1).cpu()
    return out, mag, lse


@pytest.mark.parametrize("dtype,dim,hq,hkv,page", [
    (BF16, 128, 8, 1, 16), (F16, 64, 8, 1, 64), (BF16, 64, 16, 8, 32), (F16, 128, 24, 8, 128)])
@pytest.mark.parametrize("window", [None, 2500])
@pytest.mark.parametrize("gone", [False, True])
def test_chunks_over_long_sequences(dtype, dim, hq, hkv, page, window, gone):
    # rings and rows of absent pages that wrap many times, split items, several items per CTA
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status

    c = Case([300, 37, 513], [6001, 5200, 7003], dtype=dtype, dim=dim, hq=hq, hkv=hkv, page=page,
             window=window, seed=73)
    c.there = [torch.ones(n, dtype=torch.bool) for n in c.lens]
    if gone:
        for b, at in ((0, 4200), (0, 5990), (1, 3000), (2, 6480), (2, 6999)):
            p = at // page
            c.batch.page_table[b, p] = -1
            c.there[b][p * page:(p + 1) * page] = False
    got = _attend(c)
    assert bool(device_status() & capi.TDSA_STATUS_RANGE) == gone
    _check(c, got, _torch_reference(c))


def test_many_long_items_of_two_tiles():
    c = Case([700] * 6, [2100 + 97 * i for i in range(6)], dim=64, hq=32, hkv=4, page=64, seed=74)
    c.there = [torch.ones(n, dtype=torch.bool) for n in c.lens]
    _check(c, _attend(c), _torch_reference(c))


# ------------------------------------------------------------------ scores of any size

@pytest.mark.parametrize("dtype,size", [(BF16, 300.0), (BF16, 1e4), (BF16, 1e6), (BF16, 1e12),
                                        (F16, 300.0), (F16, 5e3), (F16, 1.2e4)])
@pytest.mark.parametrize("n", [1, 8, 40])
def test_scores_of_any_size(dtype, size, n):
    # queries and keys of ``size``: scores up to 1e25, each off by 2^-17 of sum |q k|, so a row is
    # its best key's value where that leads by more; float32 holds them all
    from dsa_b200.paged import selected_attention

    c = Case([n, 3], [700, 90], dtype=dtype, dim=128, seed=80)
    c.q = (c.q.double() * size).to(dtype)
    c.qd = c.q.cuda()
    for b, length in enumerate(c.lens):
        c.k[b] = (c.k[b] * size).to(dtype).double()
        pages = c.table[b, :-(-length // c.page)].long().cuda()
        room = torch.zeros(pages.numel() * c.page, 2, 128, dtype=dtype)
        room[:length] = c.k[b].to(dtype)
        c.cache.keys[pages] = room.view(-1, c.page, 2, 128).cuda()
    out, mag, lse = c.reference()
    clear = torch.zeros(c.tokens, 8, dtype=torch.bool)
    for b, (new, length) in enumerate(zip(c.news, c.lens)):
        for i in range(new):
            t, keys = c.starts[b] + i, c.k[b][:length - new + i + 1]
            for h in range(8):
                z = keys[:, h // 4] @ c.q[t, h].double()
                best = z.topk(2).values
                room = (keys[:, h // 4].abs() @ c.q[t, h].double().abs()).max() * 2.0 ** -16
                # by so much that the second key's weight is nothing
                clear[t, h] = best[0] - best[1] > room + 40 * 128 ** 0.5
    assert clear.float().mean() > 0.8
    ind = torch.arange(700).repeat(c.tokens, 1)
    ind[ind > torch.cat([torch.arange(m - k, m) for k, m in zip(c.news, c.lens)])[:, None]] = -1
    for got, got_lse in (_attend(c), selected_attention(c.qd, c.cache, c.batch, ind.cuda(),
                                                        return_lse=True)):
        err = (got.double().cpu() - out).abs()
        u = ROUND[dtype]
        lim = (u + 2.0 ** -12) * mag + u * (1 + u) * out.abs() + 2.0 ** -24
        assert bool((err <= lim)[clear].all())
        assert bool(torch.isfinite(got).all())
        assert bool(((got_lse.double().cpu() - lse).abs() <= 2.0 ** -14 * lse.abs()).all())
