"""GPU parity of the paged key-value cache against plain 64-bit forms (tests/paged_ref.py, which also derives
the tolerances)."""
import math
import random

import pytest
import torch

import paged_ref as R
from syncopate_b200 import _lib as L
from syncopate_b200.computation.paged import page_plan, paged_append, paged_attention
from syncopate_b200.operators import PagedKVCache

pytestmark = pytest.mark.gpu
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ page_plan
def _plan_case(requests, page, max_len, max_new, seed, tokens=None, spare=5):
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, max_len)]) for _ in range(requests)]
    add = [rng.choice([-1, 0, 1, rng.randint(0, max_new)]) for _ in range(requests)]
    width = max(R.pages_of(n + max(a, 0), page) for n, a in zip(lens, add)) + 1
    held = [R.pages_of(n, page) for n in lens]
    need = sum(R.pages_of(n + a, page) - h for n, a, h in zip(lens, add, held) if a >= 0)
    pages = sum(held) + need + spare
    ids = list(range(pages))
    rng.shuffle(ids)
    at, table = 0, []
    for h in held:
        table.append(ids[at: at + h] + [-1] * (width - h))
        at += h
    free = ids[at:] + [-7] * at
    tokens = sum(max(a, 0) for a in add) + 3 if tokens is None else tokens
    return lens, add, table, free, pages - at, tokens


def _run_plan(lens, add, table, free, num_free, page, tokens, in_place=False, positions=True, status=None, stride=None):
    lens_t, table_t, free_t, num_t = ints(lens), ints(table), ints(free), ints([num_free])
    if stride:
        wide = torch.full((len(lens), stride), -3, dtype=torch.int32, device="cuda")
        wide[:, : table_t.shape[1]] = table_t
        table_t = wide[:, : table_t.shape[1]]
    slots, pos = torch.full((tokens,), 77, dtype=torch.int32, device="cuda"), torch.full((tokens,), 77, dtype=torch.int32, device="cuda")
    starts = torch.full((len(lens) + 1,), 77, dtype=torch.int32, device="cuda")
    lens_o = lens_t if in_place else torch.full_like(lens_t, 77)
    num_o = num_t if in_place else torch.full_like(num_t, 77)
    page_plan(lens_t, ints(add), table_t, free_t, num_t, page, slots, pos if positions else None, starts,
              lens_out=None if in_place else lens_o, num_free_out=None if in_place else num_o, status=status)
    if not in_place:
        assert lens_t.tolist() == lens and num_t.tolist() == [num_free]
    if stride:
        assert (wide[:, len(table[0]):] == -3).all()
    top = int(num_o)
    return slots.tolist(), pos.tolist(), starts.tolist(), lens_o.tolist(), top, table_t.tolist(), free_t.tolist()[:top]


@pytest.mark.parametrize("requests, page, max_len, max_new, tokens", [
    (1, 16, 100, 1, None), (1, 1, 3, 5, 40), (3, 16, 0, 1, None), (31, 7, 200, 3, None), (33, 64, 1000, 200, 8192),
    (257, 16, 300, 2, None), (1025, 24, 500, 9, None), (8192, 16, 40, 2, None), (5, 8, 100, 9001, None),
    (64, 16, 2000, 1999, 70001), (1024, 32, 64, 1, 1024),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_plan(requests, page, max_len, max_new, tokens, in_place):
    for seed in range(3):
        case = _plan_case(requests, page, max_len, max_new, seed, tokens)
        if tokens is not None and sum(max(a, 0) for a in case[1]) > tokens:
            continue
        status = ints([0] * 4)
        got = _run_plan(*case[:5], page, case[5], in_place=in_place, status=status, stride=len(case[2][0]) + 5)
        want = R.plan(*case[:5], page, case[5])
        assert status.tolist() == [0] * 4
        for name, g, w in zip(("slots", "positions", "starts", "lens", "num_free", "table", "free"), got, want):
            assert g == (list(w) if not isinstance(w, int) else w), name


def test_page_plan_without_positions_and_tokens():
    case = _plan_case(9, 16, 100, 0, 0, tokens=40)
    add = [min(a, 0) for a in case[1]]
    got = _run_plan(case[0], add, *case[2:5], 16, 0, positions=False)
    want = R.plan(case[0], add, *case[2:5], 16, 0)
    assert got[2:] == tuple(want[2:]) and got[0] == []


@pytest.mark.parametrize("change, code, value", [
    (dict(num_free=2), 4, None),                      # three pages needed
    (dict(tokens=10), 5, None),                       # eleven tokens
    (dict(lens=[3, -1, 40]), 5, -1),
    (dict(lens=[3, 16, 60]), 5, 60),                  # 60 + 9 tokens in rows of 64
    (dict(lens=[3, 16, 2 ** 31 - 1]), 5, 2 ** 31 - 1),
    (dict(add=[2, 2 ** 31 - 1, 2 ** 31 - 1]), 5, None),
    (dict(num_free=9), 5, None),                      # more free pages than pages
    (dict(num_free=-1), 5, None),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_plan_refuses_a_step_that_does_not_fit(change, code, value, in_place):
    base = dict(lens=[3, 16, 40], add=[2, 0, 9], num_free=3, tokens=11)
    base["add"] = [14, 1, 9] if "num_free" in change else base["add"]
    base["tokens"] = 24 if "num_free" in change else base["tokens"]
    args = {**base, **change}
    table = [[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, 4, -1]]
    free = [5, 6, 7, -1, -1, -1, -1, -1]
    status = ints([0] * 4)
    got = _run_plan(args["lens"], args["add"], table, free, args["num_free"], 16, args["tokens"], in_place=in_place, status=status)
    assert got[0] == [-1] * args["tokens"] and got[1] == [0] * args["tokens"] and got[2] == [0] * 4
    assert got[3] == args["lens"] and got[4] == args["num_free"] and got[5] == table
    words = status.tolist()
    assert words[0] == code and (value is None or words[2] == value)


def test_page_plan_gives_no_slot_on_a_page_that_does_not_exist():
    status = ints([0] * 4)
    got = _run_plan([1, 0], [1, 1], [[9], [-1]], [-5, 0, 1], 1, 16, 2, status=status)
    assert got[0] == [-1, -1] and got[1] == [1, 0] and status.tolist()[0] == 5


# ------------------------------------------------------------------ paged_append
def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


@pytest.mark.parametrize("tokens, heads, dim, page", [
    (1, 1, 64, 1), (7, 3, 128, 16), (64, 8, 128, 24), (33, 2, 256, 5), (130, 5, 48, 16), (2049, 8, 128, 64), (5, 1, 16, 3),
    (300, 16, 256, 32),
])
@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("layout", ["token", "head", "stacked"])
def test_paged_append(tokens, heads, dim, page, dtype, kept, layout):
    gen = torch.Generator().manual_seed(tokens)
    pages = R.pages_of(tokens, page) + 2
    rows = _normal(gen, tokens, 3, heads, dim, scale=3.0, dtype=dtype)
    rows[0, 1:, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 0.0], dtype=dtype)
    order = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int32)
    order[torch.rand(tokens, generator=gen) < 0.1] = -1
    order[-1] = -2 ** 31 if tokens > 1 else order[-1]
    scales = [torch.rand(heads, generator=gen) * 0.02 + 0.001 for _ in range(2)] if kept is E4 else [None, None]
    fill = _normal(gen, 2, pages, page, heads, dim).to(kept)
    if layout == "head":  # pages hold one head after the other
        buf = fill.transpose(2, 3).contiguous().cuda()
        caches = [buf[i].transpose(1, 2) for i in range(2)]
    elif layout == "stacked":  # keys and values of a page beside each other
        buf = fill.transpose(0, 1).contiguous().cuda()
        caches = [buf[:, i] for i in range(2)]
    else:
        buf = fill.cuda()
        caches = [buf[0], buf[1]]
    dev = rows.cuda()
    status = ints([0] * 4)
    paged_append(dev[:, 1], dev[:, 2], torch.cat([order, torch.zeros(3, dtype=torch.int32)]).cuda(), *caches,
                 k_scale=scales[0] if scales[0] is None else scales[0].cuda(),
                 v_scale=scales[1] if scales[1] is None else scales[1].cuda(), status=status)
    live = order >= 0
    for i in range(2):
        x = rows[:, 1 + i]
        x = R.keep(x, scales[i]) if kept is E4 else x
        word = torch.uint8 if kept is E4 else torch.int16
        want = fill[i].reshape(-1, heads, dim).clone()
        want.view(word)[order[live].long()] = x[live].view(word)
        got = caches[i].cpu().reshape(-1, heads, dim)
        if kept is E4:  # a NaN has two encodings
            assert torch.equal(torch.isnan(got.float()), torch.isnan(want.float()))
            got, want = got.float().nan_to_num(0.0), want.float().nan_to_num(0.0)
            assert torch.equal(got, want)
        else:
            assert torch.equal(got.view(word), want.view(word))
    assert status.tolist() == [0] * 4


def test_paged_append_records_a_slot_that_does_not_exist():
    k = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    caches = [torch.zeros(2, 16, 2, 64, dtype=BF, device="cuda") for _ in range(2)]
    status = ints([0] * 4)
    paged_append(k, k, ints([31, 32, 2 ** 31 - 1]), *caches, status=status)
    assert status.tolist()[0] == 5
    for c in caches:
        assert float(c.sum()) == 128.0 and (c[1, 15] == 1).all()
    paged_append(k[:0], k[:0], ints([]), *caches)


def test_every_value_is_rounded_like_a_single_rounding():
    # All 16-bit patterns through the 8-bit cache, with scales that put ties and the ends of the range on the way.
    for dtype in (BF, HF):
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(512, 1, 128)
        for scale in (1.0, 0.375, 0.0078125, 3e-5, 1000.0):
            s = torch.tensor([scale])
            caches = [torch.zeros(32, 16, 1, 128, device="cuda").to(E4) for _ in range(2)]
            paged_append(x.cuda(), x.cuda(), torch.arange(512, dtype=torch.int32, device="cuda"), *caches, k_scale=s.cuda(), v_scale=s.cuda())
            want = R.keep(x, s).float().view(-1)
            for c in caches:
                got = c.cpu().float().view(-1)
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0)), (dtype, scale)


# ------------------------------------------------------------------ paged_attention
def _make(lens, page, heads, dim, dtype, kept, seed, layout="token", scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    held = [R.pages_of(n, page) for n in lens]
    pages = sum(held) + 2
    ids = torch.randperm(pages, generator=gen).tolist()
    width, at, table = max(max(held), 1), 0, []
    for h in held:
        table.append(ids[at: at + h] + [-1] * (width - h))
        at += h
    values = _normal(gen, 2, pages, page, heads, dim, scale=60.0 if kept is E4 else scale)
    values = (values.clamp(-448, 448) if kept is E4 else values).to(kept)
    scales = [torch.rand(heads, generator=gen) * 0.01 + 0.01 for _ in range(2)] if kept is E4 else [None, None]
    if layout == "head":
        buf = values.transpose(2, 3).contiguous().cuda()
        caches = [buf[i].transpose(1, 2) for i in range(2)]
    elif layout == "stacked":
        buf = values.transpose(0, 1).contiguous().cuda()
        caches = [buf[:, i] for i in range(2)]
    else:
        buf = values.cuda()
        caches = [buf[0], buf[1]]
    return gen, table, values, caches, scales


def _cuda(x):
    return None if x is None else x.cuda()


def _compare(got, got_lse, want):
    out, lse, tol, lse_tol = want
    seen = ~torch.isnan(out)
    off = ((got.double() - out).abs() - tol)[seen]
    assert torch.isfinite(got.double()[seen]).all() and float(off.max()) <= 0, f"out off by {float(off.max())} over its bound"
    rows = ~torch.isnan(lse)
    none = lse == -math.inf
    assert (got_lse[none] == -math.inf).all()
    rows &= ~none
    if rows.any():
        assert float(((got_lse.double() - lse).abs() - lse_tol)[rows].max()) <= 0


def _check_attention(lens, news, q_heads, heads, dim, page, dtype, kept, seed=0, causal=True, window=0, layout="token", pad=0,
                     sm_scale=None, num_sms=0, scale=1.0, poison=False):
    gen, table, values, caches, scales = _make(lens, page, heads, dim, dtype, kept, seed, layout, scale)
    starts = None if news is None else [sum(news[:i]) for i in range(len(news) + 1)]
    T = (len(lens) if news is None else starts[-1]) + pad
    q = _normal(gen, T, q_heads, dim, dtype=dtype)
    sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
    if poison:  # slots that no request has, and those behind the lengths
        word = torch.uint8 if kept is E4 else torch.int16
        mask = torch.ones(values.shape[1] * page, dtype=torch.bool)
        for z, n in enumerate(lens):
            for j in range(n):
                mask[table[z][j // page] * page + j % page] = False
        for i, c in enumerate(caches):
            bad = torch.full(c.shape, 0x7F if kept is E4 else 0x7FFF if i == 0 else (0x7F80 if dtype is BF else 0x7C00), dtype=word)
            m = mask.view(-1, page)[:, :, None, None].cuda()
            c.view(word).copy_(torch.where(m, bad.cuda(), c.view(word)))
    wide = torch.randn(T, q_heads + 2, dim, generator=gen).to(dtype).cuda()  # q and out with strides of their own
    wide[:, 1:-1] = q.cuda()
    room = torch.full((T, q_heads, dim + 16), 7.0, dtype=dtype, device="cuda")
    out, lse = room[:, :, :dim], torch.full((T, q_heads), 7.0, device="cuda")
    status = ints([0] * 4)
    got = paged_attention(wide[:, 1:-1], *caches, ints(table), ints(lens), sm_scale, starts=None if news is None else ints(starts),
                          causal=causal, window=window, k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), out=out, lse=lse,
                          num_sms=num_sms, status=status)
    assert got is out and status.tolist() == [0] * 4
    assert (room[:, :, dim:] == 7).all()
    live = T - pad
    assert (out[live:] == 7).all() and (lse[live:] == 7).all()
    want = R.attention(q, values[0], values[1], table, lens, sm_scale, starts, causal, window, *scales)
    _compare(out[:live].cpu(), lse[:live].cpu(), [w[:live] for w in want])


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8, 16, 21, 40])
def test_one_token_a_request(dtype, kept, dim, group):
    _check_attention(EDGES, None, 2 * group, 2, dim, 16, dtype, kept, seed=dim + group, poison=True)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 100, 256, 1024])
@pytest.mark.parametrize("layout", ["token", "head", "stacked"])
@pytest.mark.parametrize("kept", [BF, E4])
def test_pages_and_layouts(page, layout, kept):
    _check_attention(EDGES, None, 12, 3, 128, page, BF, kept, seed=page, layout=layout, poison=True)


@pytest.mark.parametrize("dtype, kept, dim", [(BF, BF, 128), (HF, HF, 64), (HF, HF, 256), (BF, E4, 128), (HF, E4, 64), (BF, E4, 256)])
@pytest.mark.parametrize("q_heads, heads", [(4, 4), (8, 2), (10, 2), (16, 1)])
@pytest.mark.parametrize("window, causal", [(0, True), (0, False), (1, True), (37, True), (10 ** 6, True)])
def test_several_tokens_a_request(dtype, kept, dim, q_heads, heads, window, causal):
    rng = random.Random(window)
    lens = EDGES + [301, 302, 303]
    news = [rng.choice([0, 1, 1, 2, 5, 9]) for _ in lens]  # more than the length, too: rows that see nothing
    news[-1] = 70
    _check_attention(lens, news, q_heads, heads, dim, 16, dtype, kept, seed=dim, window=window, causal=causal, pad=3, poison=True)


def test_a_prompt_as_long_as_its_cache():
    _check_attention([517, 100], [517, 100], 4, 2, 128, 16, BF, BF, poison=True)


@pytest.mark.parametrize("kept", [BF, E4])
@pytest.mark.parametrize("num_sms", [0, 1, 7])
def test_long_requests_are_split_and_joined(kept, num_sms):
    _check_attention([20011, 3, 0, 9000], None, 8, 2, 128, 64, BF, kept, num_sms=num_sms)
    _check_attention([12345, 777], [3, 5], 14, 2, 64, 32, HF, E4 if kept is E4 else HF, num_sms=num_sms, window=5000)


@pytest.mark.parametrize("dim, kept, heads", [(64, E4, 4), (64, E4, 8), (64, HF, 6), (128, E4, 4), (128, E4, 3), (256, E4, 2)])
@pytest.mark.parametrize("num_sms", [0, 2])
def test_heads_taken_side_by_side(dim, kept, heads, num_sms):
    _check_attention(EDGES + [7001], None, 4 * heads, heads, dim, 16, HF, kept, num_sms=num_sms, poison=True)
    _check_attention([3000, 1, 0, 501], [5, 1, 2, 11], 6 * heads, heads, dim, 32, HF, kept, num_sms=num_sms, window=2000)


@pytest.mark.parametrize("page", [2, 5, 7, 31, 33, 4096])
def test_page_sizes_of_every_kind(page):
    _check_attention([1, page, page + 1, 3 * page - 1, 2000], None, 4, 2, 64, page, BF, BF, poison=True)


def test_the_largest_window():
    _check_attention([300, 5], [4, 9], 4, 2, 64, 16, BF, BF, window=2 ** 31 - 1)


def test_many_requests():
    rng = random.Random(1)
    _check_attention([rng.randint(0, 90) for _ in range(2100)], None, 4, 1, 64, 16, BF, BF)
    _check_attention([rng.randint(1, 700) for _ in range(300)], [rng.randint(0, 4) for _ in range(300)], 6, 2, 128, 16, BF, BF)


@pytest.mark.parametrize("sm_scale", [0.0, -0.3, 3.0])
def test_scales_of_the_scores(sm_scale):
    _check_attention([100, 700], None, 8, 2, 128, 16, BF, BF, sm_scale=sm_scale)
    _check_attention([100, 700], None, 8, 2, 128, 16, BF, E4, sm_scale=sm_scale)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_queries_of_very_different_size_over_an_8_bit_cache(dtype):
    gen, table, values, caches, scales = _make([300, 300, 300], 16, 2, 128, dtype, E4, 3)
    q = _normal(gen, 3, 8, 128) * torch.tensor([1e-4, 1.0, 300.0])[:, None, None]
    q[:, :, ::7] *= 2.0 ** -9
    q = q.to(dtype)
    lse = torch.empty(3, 8, device="cuda")
    out = paged_attention(q.cuda(), *caches, ints(table), ints([300] * 3), 0.01, k_scale=scales[0].cuda(), v_scale=scales[1].cuda(), lse=lse)
    _compare(out.cpu(), lse.cpu(), R.attention(q, values[0], values[1], table, [300] * 3, 0.01, None, True, 0, *scales))
    zero = paged_attention(torch.zeros_like(q).cuda(), *caches, ints(table), ints([300] * 3), 0.01, k_scale=scales[0].cuda(), v_scale=scales[1].cuda())
    _compare(zero.cpu(), torch.full((3, 8), math.log2(300)), R.attention(torch.zeros_like(q), values[0], values[1], table, [300] * 3, 0.01, None, True, 0, *scales))


@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_a_row_does_not_see_does_not_touch_it(dtype, kept, value, dim):
    """Keys and values that are not finite, at a position that only some of a request's rows see (the newest
    token, and the oldest one under the window)."""
    if kept is E4 and value != "nan":
        pytest.skip("the 8-bit type has no infinity")
    page, lens, news, heads, q_heads, window = 16, [100, 37, 70], [4, 3, 20], 2, 6, 33
    gen, table, values, caches, scales = _make(lens, page, heads, dim, dtype, kept, 5)
    starts = [0, 4, 7, 27]
    q = _normal(gen, 27, q_heads, dim, dtype=dtype)
    clean = R.attention(q, values[0], values[1], table, lens, 0.1, starts, True, window, *scales)
    touched = torch.zeros(27, dtype=torch.bool)
    for z, n in enumerate(lens):
        for j in (n - 2, n - news[z] - window + 2):  # seen by the rows from n - 2 on; by the first two rows
            for c, spot in ((caches[0], 3), (caches[1], 5)):
                c[table[z][j // page], j % page, :, spot] = torch.tensor(float(value)).to(kept)
            for i in range(news[z]):
                pos = n - news[z] + i
                touched[starts[z] + i] |= j <= pos and j > pos - window
    lse = torch.empty(27, q_heads, device="cuda")
    out = paged_attention(q.cuda(), *caches, ints(table), ints(lens), 0.1, starts=ints(starts), window=window,
                          k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse).cpu()
    lse = lse.cpu()
    assert 0 < int(touched.sum()) < 27
    _compare(out[~touched], lse[~touched], [w[~touched] for w in clean])
    assert not torch.isfinite(out[touched].float()).all(-1).any()


def test_pages_and_lengths_that_do_not_exist():
    lens, page = [100, 50, 70, 40], 16
    gen, table, values, caches, _ = _make(lens, page, 2, 128, BF, BF, 9)
    q = _normal(gen, 4, 8, 128, dtype=BF)
    want = R.attention(q, values[0], values[1], table, lens, 0.1)
    bad = [list(r) for r in table]
    bad[0][3] = values.shape[1]  # one behind the last page
    bad[2][4] = -1
    for lens_seen, rows in ((lens, [0, 2]), ([100, 50, 70, 7 * 16 + 1], [0, 2, 3]), ([2 ** 31 - 1, 50, 70, 40], [0, 2])):
        status, lse = ints([0] * 4), torch.empty(4, 8, device="cuda")
        out = paged_attention(q.cuda(), *caches, ints(bad), ints(lens_seen), 0.1, lse=lse, status=status).cpu()
        good = [i for i in range(4) if i not in rows]
        assert torch.isnan(out[rows].float()).all() and status.tolist()[0] == 5
        _compare(out[good], lse.cpu()[good], [w[good] for w in want])
    status = ints([0] * 4)
    out = paged_attention(q.cuda(), *caches, ints(table), ints([100, -5, 70, 40]), 0.1, status=status).cpu()
    assert (out[1] == 0).all() and status.tolist()[:3] == [5, 1, -5]
    _compare(out[[0, 2, 3]], want[1][[0, 2, 3]].float(), [w[[0, 2, 3]] for w in want])


def test_offsets_beyond_32_bits():
    # A cache of 2.2e9 elements whose last pages are in use.
    page, heads, dim = 64, 8, 128
    pages = 2 ** 31 // (page * heads * dim) + 40
    lens = [700, 65]
    gen, table, values, caches, scales = _make(lens, page, heads, dim, HF, E4, 4)
    shift = pages - values.shape[1]
    big = [torch.empty(pages, page, heads, dim, dtype=E4, device="cuda") for _ in range(2)]
    for b, c in zip(big, caches):
        b[shift:].view(torch.uint8).copy_(c.view(torch.uint8))
    far = [[x + shift if x >= 0 else x for x in r] for r in table]
    q = _normal(gen, 2, 16, dim, dtype=HF)
    lse = torch.empty(2, 16, device="cuda")
    out = paged_attention(q.cuda(), *big, ints(far), ints(lens), 0.1, k_scale=scales[0].cuda(), v_scale=scales[1].cuda(), lse=lse)
    _compare(out.cpu(), lse.cpu(), R.attention(q, values[0], values[1], table, lens, 0.1, None, True, 0, *scales))
    k = _normal(gen, 3, heads, dim, dtype=HF)
    slots = [pages * page - 1, 5, (pages - 1) * page]
    paged_append(k.cuda(), k.cuda(), ints(slots), *big, k_scale=scales[0].cuda(), v_scale=scales[1].cuda())
    for i in range(2):
        got = big[i].view(-1, heads, dim)[torch.tensor(slots, device="cuda").cpu()[0].item()].float().cpu()
        assert torch.equal(got, R.keep(k, scales[i])[0].float())
        assert torch.equal(big[i].view(-1, heads, dim)[5].float().cpu(), R.keep(k, scales[i])[1].float())


def test_same_results_at_every_call_on_any_stream():
    lens = [5000, 300, 1, 0, 17000]
    gen, table, values, caches, _ = _make(lens, 32, 2, 128, BF, BF, 2)
    q = _normal(gen, 5, 16, 128, dtype=BF).cuda()
    table_t, lens_t = ints(table), ints(lens)
    first = paged_attention(q, *caches, table_t, lens_t, 0.1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):  # calls that overlap
        outs.append(paged_attention(q, *caches, table_t, lens_t, 0.1, stream=streams[i % 3]))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


def test_two_graphs_replayed_at_once():
    lens = [4000, 700, 9000]
    gen, table, values, caches, _ = _make(lens, 16, 2, 128, BF, BF, 6)
    q = [_normal(gen, 3, 8, 128, dtype=BF).cuda() for _ in range(2)]
    table_t, lens_t = ints(table), ints(lens)
    want = [paged_attention(x, *caches, table_t, lens_t, 0.1) for x in q]
    outs, graphs = [torch.zeros_like(x) for x in q], []
    for x, out in zip(q, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(8):
                paged_attention(x, *caches, table_t, lens_t, 0.1, out=out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_rows_behind_the_last_request_without_an_output_given():
    lens, starts = [30, 40], [0, 2, 3]
    gen, table, values, caches, _ = _make(lens, 16, 2, 64, HF, HF, 8)
    q = _normal(gen, 6, 4, 64, dtype=HF)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    args = (q.cuda(), *caches, ints(table), ints(lens), 0.1)
    here = paged_attention(*args, starts=ints(starts))
    torch.cuda.synchronize()
    there = paged_attention(*args, starts=ints(starts), stream=stream)
    torch.cuda.synchronize()
    assert (here[3:] == 0).all() and torch.equal(here, there)
    want = R.attention(q, values[0], values[1], table, lens, 0.1, starts)
    _compare(here[:3].cpu(), want[1][:3].float(), [w[:3] for w in want])
    with pytest.raises(ValueError, match="8-bit"):
        paged_attention(*args, starts=ints(starts), k_scale=torch.ones(2, device="cuda"), v_scale=torch.ones(2, device="cuda"))


def test_scores_that_all_vanish_over_an_8_bit_cache():
    # A scale of zero and queries next to nothing: every key counts alike.
    gen, table, values, caches, scales = _make([37, 50], 16, 2, 128, BF, E4, 12)
    q = (_normal(gen, 5, 8, 128) * 1e-25).to(BF)
    for sm_scale in (0.0, 1.0):
        lse = torch.empty(5, 8, device="cuda")
        out = paged_attention(q.cuda(), *caches, ints(table), ints([37, 50]), sm_scale, starts=ints([0, 3, 5]), window=20,
                              k_scale=scales[0].cuda(), v_scale=scales[1].cuda(), lse=lse)
        _compare(out.cpu(), lse.cpu(), R.attention(q, values[0], values[1], table, [37, 50], sm_scale, [0, 3, 5], True, 20, *scales))


# ------------------------------------------------------------------ a run of steps
def _drive(cache, steps, q_heads, heads, dim, dtype, graph):
    """Random steps over the cache object; the same tokens are kept densely on the side."""
    gen, rng = torch.Generator().manual_seed(11), random.Random(11)
    Z, T = cache.lens.numel(), cache.slots.numel()
    layers = len(cache._k)
    dense = [[([], []) for _ in range(Z)] for _ in range(layers)]
    add = ints([0] * Z)
    qkv = torch.zeros(layers, T, q_heads + 2 * heads, dim, dtype=dtype, device="cuda")
    outs = torch.zeros(layers, T, q_heads, dim, dtype=dtype, device="cuda")
    lses = torch.zeros(layers, T, q_heads, device="cuda")

    def step():
        cache.plan(add)
        for i in range(layers):
            cache.append(qkv[i, :, q_heads: q_heads + heads], qkv[i, :, q_heads + heads:], i)
            cache.attend(qkv[i, :, :q_heads], i, out=outs[i], lse=lses[i])

    if graph:
        step()  # everything is loaded and nothing was appended
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured, stream=side):
            step()
        run = captured.replay
    else:
        run = step
    for _ in range(steps):
        left, counts = T, []
        for z in range(Z):
            n = len(dense[0][z][0])
            want = -1 if n and rng.random() < 0.15 else rng.choice([0, 1, 1, 1, rng.randint(1, 30)])
            want = min(want, left, cache.table.shape[1] * cache.page_size - n)
            counts.append(want)
            left -= max(want, 0)
        add.copy_(ints(counts))
        new = _normal(gen, layers, T, q_heads + 2 * heads, dim, dtype=dtype)
        qkv.copy_(new)
        outs.fill_(7.0)
        run()
        cache.check()
        starts = [0]
        for i in range(layers):
            at = 0
            for z, a in enumerate(counts):
                ks, vs = dense[i][z]
                if a < 0:
                    ks.clear(), vs.clear()
                for _ in range(max(a, 0)):
                    ks.append(new[i, at, q_heads: q_heads + heads])
                    vs.append(new[i, at, q_heads + heads:])
                    at += 1
                if i == 0:
                    starts.append(at)
        assert cache.starts.tolist() == starts
        lens = [len(d[0]) for d in dense[0]]
        assert cache.lens.tolist() == lens
        assert cache.positions.tolist()[: starts[-1]] == [n - max(a, 0) + j for n, a in zip(lens, counts) for j in range(max(a, 0))]
        for i in range(layers):
            width = max(max(lens), 1)
            flat = [torch.zeros(Z, width, heads, dim) for _ in range(2)]
            scales = (cache.k_scale[i], cache.v_scale[i])
            for z, pair in enumerate(dense[i]):
                for w in range(2):
                    if pair[w]:
                        flat[w][z, : lens[z]] = torch.stack(pair[w]).float()
            if scales[0] is not None:
                scales = tuple(s.cpu() for s in scales)
                flat = [R.keep(f.view(-1, heads, dim), s).view(f.shape) for f, s in zip(flat, scales)]
            else:
                flat = [f.to(dtype) for f in flat]
            want = R.attention(new[i, :, :q_heads], flat[0], flat[1], [[z] for z in range(Z)], lens, dim ** -0.5, starts, True, 0,
                               *scales)
            n = starts[-1]
            if n:
                _compare(outs[i, :n].cpu(), lses[i, :n].cpu(), [w[:n] for w in want])
            assert (outs[i, n:] == 7).all()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kept", [None, E4])
def test_a_run_of_steps(graph, kept):
    heads, q_heads, dim, layers = 2, 8, 128, 2
    scales = {} if kept is None else dict(k_scale=torch.rand(layers, heads) * 0.01 + 0.01, v_scale=torch.rand(layers, heads) * 0.01 + 0.01)
    cache = PagedKVCache(200, 8, heads, dim, 9, 150, 64, layers=layers, dtype=BF, cache_dtype=kept, device="cuda:0", **scales)
    cache.kv.view(torch.uint8).fill_(0xFF)  # NaN in every slot that nothing was written to
    _drive(cache, 25, q_heads, heads, dim, BF, graph)


def test_a_step_that_does_not_fit_is_told_and_changes_nothing():
    cache = PagedKVCache(3, 16, 1, 64, 2, 64, 40, dtype=HF)
    x = torch.randn(40, 1, 64, device="cuda").to(HF)
    cache.plan(ints([20, 1]))
    cache.append(x, x)
    kept = cache.kv.clone()
    cache.check()
    cache.plan(ints([20, 16]))
    cache.append(x, x)
    out = torch.full_like(x, 7.0)
    cache.attend(x, out=out)
    with pytest.raises(L.SynError) as e:
        cache.check()
    assert e.value.code == L.SYN_ERR_NO_PAGES
    assert cache.lens.tolist() == [20, 1] and cache.num_free.tolist() == [0]
    assert torch.equal(cache.kv.view(torch.int16), kept.view(torch.int16)) and (out == 7).all()
    cache.check()  # told once
    cache.plan(ints([-1, 16]))  # the first request makes room
    cache.check()
    assert cache.lens.tolist() == [0, 17] and cache.num_free.tolist() == [1]


@pytest.mark.parametrize("kept", [BF, E4])
@pytest.mark.parametrize("window", [0, 1, 7, 40, 200])
@pytest.mark.parametrize("past", [1, 3, 5, 9, 60, 2 ** 31 - 1 - 112])
def test_new_tokens_behind_the_row_of_the_table(kept, window, past):
    """Request 0 says that it is `past` tokens longer than its row of the table has room for: its tokens from there on
    need a key that no page holds, those before are where they say they are."""
    page, room, news, heads, q_heads, dim = 16, 112, [5, 3], 2, 8, 128
    gen, table, values, caches, scales = _make([room, 50], page, heads, dim, BF, kept, 31)
    q = _normal(gen, 8, q_heads, dim, dtype=BF)
    there = max(0, news[0] - past)  # tokens before the end of the table
    rows = list(range(there)) + [5, 6, 7]
    for causal in (True, False) if window == 0 else (True,):
        status, lse = ints([0] * 4), torch.empty(8, q_heads, device="cuda")
        out = paged_attention(q.cuda(), *caches, ints(table), ints([room + past, 50]), 0.1, starts=ints([0, 5, 8]), causal=causal,
                              window=window, k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse, status=status).cpu()
        assert status.tolist()[:2] == [5, 0]
        seen = rows if causal else rows[there:]
        gone = [i for i in range(8) if i not in seen]
        assert torch.isnan(out[gone].float()).all() and torch.isnan(lse.cpu()[gone]).all()
        want = R.attention(q[rows], values[0], values[1], table, [room, 50], 0.1, [0, there, there + 3], causal, window, *scales)
        at = [rows.index(i) for i in seen]
        _compare(out[seen], lse.cpu()[seen], [w[at] for w in want])


@pytest.mark.parametrize("kept", [BF, E4])
@pytest.mark.parametrize("window, causal", [(0, True), (0, False), (1, True), (9, True)])
def test_fewer_rows_than_the_requests_say(kept, window, causal):
    # Request 1 has two of its five rows behind the end of q, request 2 all of them: the rows that are there stay in place.
    lens, starts, heads, q_heads, dim = [40, 70, 33], [0, 4, 9, 11], 2, 8, 128
    gen, table, values, caches, scales = _make(lens, 16, heads, dim, BF, kept, 32)
    q = _normal(gen, 11, q_heads, dim, dtype=BF)
    want = R.attention(q, values[0], values[1], table, lens, 0.1, starts, causal, window, *scales)
    status, lse = ints([0] * 4), torch.empty(7, q_heads, device="cuda")
    out = paged_attention(q[:7].cuda(), *caches, ints(table), ints(lens), 0.1, starts=ints(starts), causal=causal, window=window,
                          k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse, status=status)
    assert status.tolist()[0] == 5
    _compare(out.cpu(), lse.cpu(), [w[:7] for w in want])


# (bits below the first key, the same a little lower), both of them numbers of the 8-bit type
DEPTHS = [(8, 9), (14, 15), (18, 20), (22, 24), (26, 28), (40, 44), (72, 80)]


@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("dim, group", [(64, 4), (64, 40), (128, 8), (128, 16), (128, 32), (256, 8), (256, 16)])
@pytest.mark.parametrize("depth", DEPTHS)
def test_weights_far_below_the_largest(dtype, kept, dim, group, depth):
    """One key takes the weight and its value is 0, so that the output is made of the weights that are 8 to 160 bits
    smaller: each has to count with its 16 bits, however small, and some that nobody sees are NaN."""
    sm_scale, lens, news = 0.97 * math.log(2.0), [40, 1500], [2, 1]
    gen, table, values, caches, scales = _make(lens, 16, 1, dim, dtype, kept, sum(depth))
    k, v = [x.float() for x in values]
    k[..., 0] = -torch.tensor(depth, dtype=torch.float32)[torch.randint(2, k.shape[:-1], generator=gen)]
    v = (1.0 + 0.25 * _normal(gen, *v.shape)).clamp(0.25, 1.75) * (100.0 if kept is E4 else 8192.0)
    for z in range(2):
        k[table[z][0], 3, 0, 0] = 0.0
        v[table[z][0], 3] = 0.0
    k, v = k.to(kept), v.to(kept)
    if kept is E4:
        scales = [torch.ones(1), torch.full((1,), 81.92)]
    hidden = v.clone()  # the newest token of request 0 is hidden from the one before
    hidden.view(torch.uint8 if kept is E4 else torch.int16)[table[0][39 // 16], 39 % 16, 0, dim // 2] = 0x7F if kept is E4 else 0x7FFF
    # Only the first dimension of a query counts, so that scores are products without a sum; four sizes of them.
    q = torch.zeros(3, group, dim, dtype=dtype)
    q[:, :, 0] = torch.tensor([1.0, 0.5, 2.0, 1.0]).repeat(-(-group // 4))[:group].to(dtype)
    starts, args = [0, 2, 3], (table, lens, sm_scale, [0, 2, 3], True, 0, *scales)
    want, want_lse = R.attention(q, k, v, *args)[:2]
    # An exponent of up to X bits: sm_scale, log2 e, their product, the key's scale and the difference from the reference
    # are rounded to 2^-24 each: 5 X ln 2 2^-24 in the weight.  exp2 and the factors of rescaling and joining: 2^-19.
    # The weight in the product: 2^-16.  Sums of n terms: n 2^-23 in numerator and denominator.
    X = 2 * depth[1] * 0.97
    rel = 5 * X * math.log(2.0) * 2.0 ** -24 + 2.0 ** -19 + 2.0 ** -16 + (max(lens) + 64) * 2.0 ** -23
    # A weight below 2^-126, the least normal number of 32 bits, counts as 0: each of n misses at most 2^-126 |v| of a sum
    # that is 1 or more.
    bound = want.abs() * rel + max(lens) * 2.0 ** -126 * float(v.float().max()) * (81.92 if kept is E4 else 1.0)  # values are not negative
    fi = torch.finfo(dtype)
    bound = bound + fi.eps / 2 * (want.abs() + bound) + fi.smallest_normal * fi.eps / 2
    word = torch.uint8 if kept is E4 else torch.int16
    for num_sms in (0, 1):
        for values_seen, last in ((v, 3), (hidden, 1)):
            lse = torch.empty(3, group, device="cuda")
            caches[0].view(word).copy_(k.view(word))
            caches[1].view(word).copy_(values_seen.view(word))
            out = paged_attention(q.cuda(), *caches, ints(table), ints(lens), sm_scale, starts=ints(starts), num_sms=num_sms,
                                  k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse).cpu().double()
            rows = [0, 1, 2] if last == 3 else [0, 2]
            off = float(((out - want).abs() - bound)[rows].max())
            assert off <= 0, f"out off by {off} over its bound, {float(((out - want).abs() / want.abs())[rows].max())} of it"
            assert float((lse.cpu().double() - want_lse).abs().max()) <= 2.0 ** -19 + max(lens) * 2.0 ** -24


@pytest.mark.parametrize("kept", [BF, E4])
@pytest.mark.parametrize("rows", [0, 1, 3, 700])
def test_paged_append_records_tokens_without_a_row(kept, rows):
    gen = torch.Generator().manual_seed(rows)
    x = _normal(gen, rows, 2, 64, dtype=BF).cuda()
    scales = dict(k_scale=torch.ones(2, device="cuda"), v_scale=torch.ones(2, device="cuda")) if kept is E4 else {}
    slots = list(range(rows)) + [-1] * 900
    caches = [torch.zeros(100, 16, 2, 64, device="cuda").to(kept) for _ in range(2)]
    for live in (None, rows, rows + 899):
        at = list(slots)
        if live is not None:
            at[live] = 1599
        status = ints([0] * 4)
        paged_append(x, x, ints(at), *caches, **scales, all_slots=True, status=status)
        assert status.tolist()[:3] == ([0, 0, 0] if live is None else [5, live, 1599])
        for c in caches:
            flat = c.float().view(-1, 2, 64)
            assert torch.equal(flat[:rows], x.to(kept).float()) and (flat[rows:] == 0).all()


def test_a_step_with_fewer_rows_than_it_planned_is_told():
    cache = PagedKVCache(8, 16, 1, 64, 2, 64, 40, dtype=HF)
    x = torch.randn(40, 1, 64, device="cuda").to(HF)
    cache.plan(ints([20, 1]))
    cache.append(x[:21], x[:21])
    cache.check()
    cache.plan(ints([1, 1]))
    cache.append(x[:1], x[:1])
    with pytest.raises(L.SynError) as e:
        cache.check()
    assert e.value.code == L.SYN_ERR_BAD_INDEX


@pytest.mark.parametrize("size, sm_scale", [(1e16, 1e-33), (1e16, -1e-33), (1e18, 1e-37)])
def test_the_smallest_scales_of_the_scores(size, sm_scale):
    lens, news = [100, 700], [3, 2]
    gen, table, values, caches, _ = _make(lens, 16, 2, 128, BF, BF, 43)
    q, k = (_normal(gen, 5, 8, 128) * size).to(BF), (values[0].float() * size).to(BF)
    caches[0].copy_(k)
    lse = torch.empty(5, 8, device="cuda")
    out = paged_attention(q.cuda(), *caches, ints(table), ints(lens), sm_scale, starts=ints([0, 3, 5]), window=300, lse=lse)
    _compare(out.cpu(), lse.cpu(), R.attention(q, k, values[1], table, lens, sm_scale, [0, 3, 5], True, 300))


@pytest.mark.parametrize("power, sm_scale", [(0, 0.09), (100, 0.09 * 2.0 ** -100), (113, 0.09 * 2.0 ** -113), (120, 0.09 * 2.0 ** -120)])
def test_the_largest_queries_over_an_8_bit_cache(power, sm_scale):
    lens = [100, 700]
    gen, table, values, caches, scales = _make(lens, 16, 2, 128, BF, E4, 42)
    q = (_normal(gen, 2, 8, 128) * 2.0 ** power).to(BF)
    lse = torch.empty(2, 8, device="cuda")
    out = paged_attention(q.cuda(), *caches, ints(table), ints(lens), sm_scale, k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse)
    _compare(out.cpu(), lse.cpu(), R.attention(q, values[0], values[1], table, lens, sm_scale, None, True, 0, *scales))


def test_the_cache_knows_its_device():
    cache = PagedKVCache(4, 16, 1, 64, 2, 64, 8, device="cuda")
    assert cache.device == cache.kv.device == torch.device("cuda", torch.cuda.current_device())


@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("dim, q_heads, heads", [(64, 8, 4), (128, 6, 2), (128, 32, 1), (256, 16, 1)])
def test_scores_that_spread_over_many_powers_of_two(dtype, kept, dim, q_heads, heads):
    # Scores of 10 and more on either side: most steps hold weights that halves have no place for.
    _check_attention([2000, 1, 333, 0, 64], None, q_heads, heads, dim, 16, dtype, kept, seed=51, sm_scale=6.0 * dim ** -0.5, poison=True)
    _check_attention([2000, 700, 90], [3, 9, 2], q_heads, heads, dim, 16, dtype, kept, seed=52, sm_scale=6.0 * dim ** -0.5, window=450,
                     num_sms=1, poison=True)


@pytest.mark.parametrize("dtype, kept", [(BF, BF), (HF, HF), (BF, E4)])
@pytest.mark.parametrize("rows", [1, 2, 4])
@pytest.mark.parametrize("window", [0, 6])
def test_rows_that_are_left_of_a_request_do_not_see_its_newer_tokens(dtype, kept, rows, window):
    # Five new tokens, of which q has the first few; what only the others see is NaN.
    length, heads, q_heads, dim = 53, 2, 8, 64
    gen, table, values, caches, scales = _make([length], 16, heads, dim, dtype, kept, 61)
    q = _normal(gen, 5, q_heads, dim, dtype=dtype)
    want = R.attention(q, values[0], values[1], table, [length], 0.1, [0, 5], True, window, *scales)
    for c in caches:
        for j in range(length - 5 + rows, length):
            c[table[0][j // 16], j % 16] = torch.full((heads, dim), math.nan).to(kept)
    lse = torch.empty(rows, q_heads, device="cuda")
    out = paged_attention(q[:rows].cuda(), *caches, ints(table), ints([length]), 0.1, starts=ints([0, 5]), window=window,
                          k_scale=_cuda(scales[0]), v_scale=_cuda(scales[1]), lse=lse)
    _compare(out.cpu(), lse.cpu(), [w[:rows] for w in want])
