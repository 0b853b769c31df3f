"""Token-paged 8-bit cache on the GPU: append, book-keeping and attention against plain 64-bit counterparts."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

E_RANGE, E_NOMEM = -4, -5


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_cache(lens, page, hkv, layers=1, extra=2, spare_rows=0, seed=0, per_row=None, poison=True):
    """A cache with lens[i] tokens of random codes in row i, pages scattered; what lies behind a sequence's end, in free
    pages and in their scales, is NaN codes and huge scales unless poison is off."""
    import magi_b200 as mb
    rng = np.random.RandomState(seed)
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + extra
    c = mb.TokenPagedKVCache(layers, n_pages, page, hkv, len(lens) + spare_rows, per_row or max(counts + [1]))
    order, at = rng.permutation(n_pages), 0
    table, refs = np.full((c.max_seqs, c.max_pages_per_seq), -1, np.int32), np.zeros(n_pages, np.int32)
    shape = (layers, n_pages, hkv, page, 128)
    codes = [R.to_code(np.clip(rng.randn(*shape) * 90, -448, 448)) for _ in range(2)]
    scales = [2.0 ** rng.randint(-9, -4, shape[:3]) for _ in range(2)]
    used = np.zeros(n_pages, bool)
    for i, n in enumerate(counts):
        ids = order[at:at + n]
        at += n
        table[i, :n], refs[ids], used[ids] = ids, 1, True
        if n and lens[i] % page and poison:
            for x in codes:
                x[:, ids[-1], :, lens[i] % page:] = 0x7f
    if poison:
        for x, s in zip(codes, scales):
            x[:, ~used], s[:, ~used] = 0xff, 2.0 ** 60
    for t, x in ((c.k8, codes[0]), (c.v8, codes[1])):
        t.view(torch.uint8).copy_(torch.from_numpy(x))
    for t, x in ((c.k_scale, scales[0]), (c.v_scale, scales[1]), (c.page_table, table), (c.page_refs, refs)):
        t.copy_(torch.from_numpy(x))
    c.seq_lens[:len(lens)] = i32(list(lens))
    return c


def strided_bf16(t, h, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h + pad, 128 + 8 * pad, generator=g).to(torch.bfloat16).cuda()
    return x[:, :h, :128]


def status():
    import magi_b200 as mb
    return mb.Context.get().status()


def check_attn(c, q, seqs, cu, **kw):
    import magi_b200 as mb
    total, hq, _ = q.shape
    n_q = [b - a for a, b in zip(cu, cu[1:])]
    out = torch.full((total, hq, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    single = all(n == 1 for n in n_q) and total == len(seqs)
    got, lse = mb.paged_attn(q, c, kw.pop("layer", 0), i32(seqs), None if single else i32(cu), max_q=max(n_q + [1]), out=out, **kw)
    torch.cuda.synchronize()
    assert got is out and status() == 0
    kw.pop("softmax_scale", None) if kw.get("softmax_scale") is None else None
    ref, ref_l, tol, tol_l = R.attention(R.Books(c), 0, q.double().cpu().numpy(), seqs, cu, c.n_kv_heads,
                                         scale=kw.get("softmax_scale"), causal=kw.get("causal", True), window=kw.get("window", 0))
    o, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    owned = np.zeros(total, bool)
    owned[cu[0]:cu[-1]] = True
    assert (o[~owned] == 7.0).all(), "rows that no entry owns were written"
    err = np.abs(o - ref)[owned]
    assert np.array_equal(np.isnan(o[owned]), np.isnan(ref[owned]))
    fine = np.isfinite(ref[owned])
    assert (err[fine] <= tol[owned][fine]).all(), f"worst {np.nanmax(err / np.maximum(tol[owned], 1e-30))} of the tolerance"
    both = np.isneginf(ref_l[owned]) == np.isneginf(l[owned])
    assert both.all()
    fl = np.isfinite(ref_l[owned])
    assert (np.abs(l - ref_l)[owned][fl] <= tol_l[owned][fl]).all()
    return o


# ---------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,hkv", [(6, 1), (8, 8), (48, 8), (16, 1), (20, 1), (6, 2)])
def test_one_token_per_sequence(page, hq, hkv):
    lens = [1, 0, 15, 16, 17, 127, 128, 129, 255, 257, 640, 1000]
    c = make_cache(lens, page, hkv, seed=page + hq)
    check_attn(c, strided_bf16(len(lens), hq, 3), list(range(len(lens))), list(range(len(lens) + 1)))


@pytest.mark.parametrize("page,hq,hkv,window,causal", [(16, 6, 1, 0, True), (64, 48, 8, 0, True), (32, 6, 2, 5, True), (128, 8, 2, 100, True),
                                                       (64, 6, 1, 0, False), (16, 12, 2, 129, False), (32, 24, 8, 1, True)])
def test_several_tokens_per_sequence(page, hq, hkv, window, causal):
    # more rows than keys, rows at every offset of a 128-key tile, an entry without rows
    lens, n_q = [0, 3, 130, 256, 300, 77, 391], [4, 5, 2, 9, 17, 0, 64]
    c = make_cache(lens, page, hkv, seed=page)
    cu = np.concatenate([[0], np.cumsum(n_q)]).tolist()
    q = strided_bf16(cu[-1] + 3, hq, 5, pad=1)  # three rows that no entry owns
    check_attn(c, q, list(range(len(lens))), cu, window=window, causal=causal)


@pytest.mark.parametrize("page,hq,hkv", [(64, 48, 8), (16, 6, 1), (128, 4, 4)])
def test_prompts(page, hq, hkv):
    lens, n_q = [513, 200, 333], [513, 129, 40]
    c = make_cache(lens, page, hkv, seed=1)
    check_attn(c, strided_bf16(sum(n_q), hq, 9), [0, 1, 2], np.concatenate([[0], np.cumsum(n_q)]).tolist())


def test_long_context_is_split_and_joined():
    c = make_cache([40003, 129], 64, 1, seed=2)
    check_attn(c, strided_bf16(2, 6, 1), [0, 1], [0, 1, 2])
    check_attn(c, strided_bf16(5, 6, 2), [0, 1], [0, 3, 5], softmax_scale=0.3)


def test_the_same_sequence_twice_and_an_order_of_their_own():
    c = make_cache([70, 400, 129], 32, 2, seed=4)
    o = check_attn(c, strided_bf16(4, 4, 8)[[0, 1, 0, 2]], [2, 1, 2, 0], [0, 1, 2, 3, 4])
    assert np.array_equal(o[0], o[2])


def test_sharp_softmax_and_pages_of_very_different_scale():
    """Scores of +-100s and V scales 2^40 apart: the weights of the small pages must not vanish where they win."""
    c = make_cache([300], 16, 1, seed=6)
    used = c.page_table[0, :19].long()
    c.v_scale[0, used, 0] = torch.tensor([2.0 ** (40 * ((i % 3) - 1)) for i in range(19)], device="cuda")
    c.k_scale[0, used, 0] = 2.0 ** -3
    check_attn(c, strided_bf16(1, 6, 11), [0], [0, 1])
    # one page wins by far, and it is one of the small ones
    import magi_b200 as mb
    c.k8.view(torch.uint8)[0, used, 0] = 0x38  # every key is all ones
    c.k_scale[0, used, 0] = 2.0 ** -10
    c.k_scale[0, used[3], 0] = 1.0
    c.v_scale[0, used, 0] = 2.0 ** 20
    c.v_scale[0, used[3], 0] = 2.0 ** -20
    q = torch.full((1, 6, 128), 2.0, dtype=torch.bfloat16, device="cuda")
    check_attn(c, q, [0], [0, 1])


def test_nan_and_infinity_where_nothing_looks():
    """NaN in later tokens than a row may see stays out of it and reaches the rows that do see it."""
    c = make_cache([260], 32, 1, seed=7)
    ids = c.page_table[0].long()
    page, off = int(ids[250 // 32]), 250 % 32
    c.v8.view(torch.uint8)[0, page, 0, off, 5] = 0x7f   # V of position 250, channel 5
    page2, off2 = int(ids[255 // 32]), 255 % 32
    c.k8.view(torch.uint8)[0, page2, 0, off2] = 0xff     # K of position 255
    o = check_attn(c, strided_bf16(16, 6, 12), [0], [0, 16])   # positions 244 .. 259
    assert np.isfinite(o[:6]).all() and np.isnan(o[6:11, :, 5]).all() and np.isfinite(o[6:11, :, 6:]).all() and np.isnan(o[11:]).all()


def test_nan_and_infinite_queries_stay_in_their_rows():
    c = make_cache([200], 64, 1, seed=8)
    q = strided_bf16(3, 6, 13).clone()
    import magi_b200 as mb
    clean, _ = mb.paged_attn(q, c, 0, i32([0]), i32([0, 3]), max_q=3)
    q[0, 2, 17] = math.nan
    q[1, 4, 3] = math.inf
    out, lse = mb.paged_attn(q, c, 0, i32([0]), i32([0, 3]), max_q=3)
    bad = torch.zeros(3, 6, dtype=torch.bool, device="cuda")
    bad[0, 2] = bad[1, 4] = True
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("n_q,window", [(2, 0), (2, 20), (5, 0), (5, 9), (40, 0), (40, 30)])
def test_nan_values_reach_only_the_rows_that_see_them(n_q, window):
    """In every form (12, 30 and 240 rows of the kv head), with NaN codes on both sides of what the rows see."""
    n = 300
    c = make_cache([n], 32, 1, seed=n_q)
    ids = c.page_table[0].long()
    spots = [(n - 1, 3), (n - 2, 64), (n - 1, 127), (n - n_q - 15, 70), (n - n_q, 31), (n - 130, 9)]  # (position, channel)
    for at, ch in spots:
        c.v8.view(torch.uint8)[0, int(ids[at // 32]), 0, at % 32, ch] = 0xff if ch & 1 else 0x7f
    o = check_attn(c, strided_bf16(n_q, 6, 17), [0], [0, n_q], window=window)
    for at, ch in spots:
        for t in range(n_q):
            pos = n - n_q + t
            assert np.isnan(o[t, :, ch]).all() == (at <= pos and (window == 0 or at > pos - window)), (at, ch, t)


# More units than blocks, so that every block begins and ends several; short ones, whose tiles are all at a border.
@pytest.mark.parametrize("n,hq,hkv,q_hi,len_hi,window", [(900, 8, 2, 1, 300, 0), (900, 8, 2, 1, 300, 40), (700, 12, 2, 5, 400, 0), (700, 12, 2, 5, 400, 130),
                                                         (260, 6, 1, 300, 420, 0), (260, 6, 1, 300, 420, 150), (150, 21, 3, 70, 200, 3)])
def test_many_short_units(n, hq, hkv, q_hi, len_hi, window):
    rng = np.random.RandomState(n + window)
    lens = rng.randint(0, len_hi + 1, n).tolist()
    n_q = [1] * n if q_hi == 1 else rng.randint(0, q_hi + 1, n).tolist()
    c = make_cache(lens, 64 if window else 16, hkv, seed=n)
    cu = np.concatenate([[0], np.cumsum(n_q)]).tolist()
    check_attn(c, strided_bf16(cu[-1], hq, 19), rng.permutation(n).tolist(), cu, window=window)


@pytest.mark.parametrize("n_q,hq", [(1, 6), (4, 6), (8, 6)])
def test_one_long_sequence_among_many_short_ones(n_q, hq):
    """A block's part then reaches hundreds of short entries, some of them without rows."""
    rng = np.random.RandomState(n_q)
    n = 1024
    lens = rng.randint(n_q, 20, n).tolist()
    rows = np.where(rng.rand(n) < 0.4, 0, n_q).tolist()
    lens[300], rows[300] = 200000, n_q
    c = make_cache(lens, 128, 1, seed=n_q)
    cu = np.concatenate([[0], np.cumsum(rows)]).tolist()
    check_attn(c, strided_bf16(cu[-1], hq, 29), list(range(n)), cu)


@pytest.mark.parametrize("n_q", [1, 4, 8])
def test_much_work_and_many_short_entries(n_q):
    """100 entries of one long sequence, the same rows, between 924 short ones: a block's part is then worth hundreds of those."""
    import magi_b200 as mb
    rng = np.random.RandomState(n_q)
    lens = [131072 - 5] + rng.randint(n_q, 20, 924).tolist()
    c = make_cache(lens, 128, 1, seed=n_q)
    q = strided_bf16(925 * n_q, 6, 31)
    order = np.concatenate([np.zeros(100, np.int64), np.arange(1, 925)])
    rng.shuffle(order)
    order[:500] = np.sort(order[:500])  # long ones in a row, and long ones apart
    rows = (order[:, None] * n_q + np.arange(n_q)).reshape(-1)
    got, _ = mb.paged_attn(q[torch.from_numpy(rows).cuda()], c, 0, i32(order.tolist()), i32((np.arange(1025) * n_q).tolist()), max_q=n_q)
    ref, _, tol, _ = R.attention(R.Books(c), 0, q.double().cpu().numpy(), list(range(925)), (np.arange(926) * n_q).tolist(), 1)
    assert status() == 0
    assert (np.abs(got.double().cpu().numpy() - ref[rows]) <= tol[rows]).all()


@pytest.mark.parametrize("hq,hkv,n_q", [(21, 3, 2), (21, 3, 4), (21, 3, 60), (5, 1, 6), (13, 1, 11), (31, 1, 1), (31, 1, 9), (33, 1, 1), (257, 1, 3)])
def test_groups_that_are_no_power_of_two(hq, hkv, n_q):
    c = make_cache([n_q + 150, n_q], 32, hkv, seed=hq)
    check_attn(c, strided_bf16(2 * n_q, hq, 23), [0, 1], [0, n_q, 2 * n_q])


def test_scores_that_grow_from_tile_to_tile():
    """Every tile asks for a new reference, by less and by more than what a weight has room for."""
    for step in (0.5, 2.0, 3.9, 9.0, 40.0):
        n = 1500
        c = make_cache([n], 64, 1, seed=31)
        ids = c.page_table[0].long()
        c.k8.view(torch.uint8).zero_()
        c.k_scale.fill_(2.0 ** -20)
        for page, i in enumerate(ids[:-(-n // 64)].tolist()):
            c.k8.view(torch.uint8)[0, i, 0, :, 0] = 0x38          # 1.0 in channel 0, times the page's scale
            c.k8.view(torch.uint8)[0, i, 0, :, 1] = (torch.arange(64, device="cuda") % 8 + 0x30).to(torch.uint8)
            c.k_scale[0, i, 0] = 2.0 ** (page // 2 - 6)           # doubles from tile to tile
        q = torch.zeros(40, 6, 128, dtype=torch.bfloat16, device="cuda")
        q[:, :, 0] = step
        q[:, :, 1] = torch.linspace(-1, 1, 40, device="cuda").to(torch.bfloat16)[:, None]
        for m in (1, 5, 40):
            check_attn(c, q[:m], [0], [0, m])


def test_queries_of_any_size():
    c = make_cache([150], 64, 1, seed=9)
    q = strided_bf16(6, 6, 14) * torch.tensor([1e-30, 0.0, 1e-3, 30.0, 1.0, 1e-38], device="cuda")[:, None, None].to(torch.bfloat16)
    check_attn(c, q, [0], [0, 6])


def test_layers_and_out_and_strides():
    import magi_b200 as mb
    c = make_cache([100, 33], 32, 2, layers=3, seed=10)
    q = strided_bf16(2, 4, 15, pad=2)
    books = R.Books(c)
    for layer in range(3):
        wide = torch.zeros(4, 7, 144, dtype=torch.bfloat16, device="cuda")
        out, lse = mb.paged_attn(q, c, layer, i32([0, 1]), out=wide[:, 1:5, 8:136])
        ref, _, tol, _ = R.attention(books, layer, q.double().cpu().numpy(), [0, 1], [0, 1, 2], 2)
        assert (np.abs(out[:2].double().cpu().numpy() - ref) <= tol).all()
        wide[:2, 1:5, 8:136] = 0
        assert (wide == 0).all()
        none = mb.paged_attn(q, c, layer, i32([0, 1]), return_lse=False)
        assert none[1] is None and torch.equal(none[0], mb.paged_attn(q, c, layer, i32([0, 1]))[0])


def test_results_do_not_change_from_call_to_call():
    import magi_b200 as mb
    c = make_cache([5000, 77, 1300], 64, 2, seed=20)
    q = strided_bf16(3, 12, 21)
    first = mb.paged_attn(q, c, 0, i32([0, 1, 2]))
    for _ in range(5):
        again = mb.paged_attn(q, c, 0, i32([0, 1, 2]))
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_streams_at_once():
    import magi_b200 as mb
    c = make_cache([9000, 500], 64, 2, layers=2, seed=22)
    q = strided_bf16(2, 12, 23)
    want = [mb.paged_attn(q, c, layer, i32([0, 1])) for layer in range(2)]
    side = [torch.cuda.Stream() for _ in range(2)]
    seqs = i32([0, 1])
    torch.cuda.synchronize()
    got = [[mb.paged_attn(q, c, layer, seqs, stream=side[layer]) for layer in range(2)] for _ in range(20)]
    torch.cuda.synchronize()
    for pair in got:
        for w, g in zip(want, pair):
            assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])


def test_a_table_that_points_nowhere_is_reported():
    import magi_b200 as mb
    c = make_cache([300], 64, 1, seed=24)
    c.page_table[0, 2] = 10 ** 6
    mb.paged_attn(strided_bf16(1, 6, 1), c, 0, i32([0]))
    assert status() == E_RANGE
    mb.paged_attn(strided_bf16(1, 6, 1), c, 0, i32([5]))
    assert status() == E_RANGE and status() == 0


# ---------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hkv", [1, 3, 8])
def test_append_matches_the_definition(page, hkv):
    rng = np.random.RandomState(page + hkv)
    lens, new = [0, 1, 15, 16, 130, 255, 7, 64], [1, 16, 1, 3, 300, 1, 0, 129]
    total = [a + b for a, b in zip(lens, new)]
    c = make_cache(total, page, hkv, layers=2, seed=1)
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    size = np.exp(2 * rng.randn(cu[-1], 1, 1))
    k, v = [torch.from_numpy(rng.randn(cu[-1], hkv, 128) * size).to(torch.bfloat16).cuda() for _ in range(2)]
    wide = torch.zeros(cu[-1], hkv + 1, 264, dtype=torch.bfloat16, device="cuda")
    wide[:, :hkv, :128], wide[:, :hkv, 136:] = k, v
    books = R.Books(c)
    for i in range(len(lens)):
        books.append(1, i, lens[i], k[cu[i]:cu[i + 1]].double().cpu().numpy(), v[cu[i]:cu[i + 1]].double().cpu().numpy())
    c.append(1, i32(list(range(len(lens)))), i32(lens), wide[:, :hkv, :128], wide[:, :hkv, 136:], i32(cu), max_new=max(new))
    torch.cuda.synchronize()
    assert status() == 0 and books.same(c) is None, books.same(c)


def test_token_by_token():
    """Scales that grow many times over; the last page is written token after token."""
    rng = np.random.RandomState(3)
    c = make_cache([0, 5], 32, 2, seed=2, extra=8, per_row=4)
    books = R.Books(c)
    for step in range(70):
        size = 2.0 ** rng.randint(-30, 30)
        k, v = [torch.from_numpy(rng.randn(2, 2, 128) * size).to(torch.bfloat16).cuda() for _ in range(2)]
        starts = c.reserve(i32([1, 0]), i32([1, 1]))
        assert starts.tolist() == books.reserve([1, 0], [1, 1])
        c.append(0, i32([1, 0]), starts, k, v)
        for i, s in enumerate((1, 0)):
            books.append(0, s, books.lens[s] - 1, k[i:i + 1].double().cpu().numpy(), v[i:i + 1].double().cpu().numpy())
    assert status() == 0 and books.same(c) is None, books.same(c)


def test_append_of_unusual_values():
    c = make_cache([0], 16, 1, seed=2, extra=4, per_row=2)
    c.reserve(i32([0]), i32([20]))
    books = R.Books(c)
    x = torch.zeros(20, 1, 128)
    x[0, 0, :6] = torch.tensor([math.nan, math.inf, -math.inf, 3.0, -448.0, 1e-30])
    x[1:15, 0] = torch.randn(14, 128) * 100
    x[16, 0, :4] = torch.tensor([1e38, -3e38, 1e-38, 0.0])    # beyond 448 * 2^60: the scale's end, saturated
    x = x.to(torch.bfloat16).cuda()
    tiny = (torch.randn(20, 1, 128) * 1e-30).to(torch.bfloat16).cuda()  # below the smallest scale: zeros
    c.append(0, i32([0]), i32([0]), x, tiny, i32([0, 20]), max_new=20)
    books.append(0, 0, 0, x.double().cpu().numpy(), tiny.double().cpu().numpy())
    assert status() == 0 and books.same(c) is None, books.same(c)
    assert float(c.k_scale[0, int(c.page_table[0, 1]), 0]) == 2.0 ** 60 and float(c.v_scale[0, int(c.page_table[0, 0]), 0]) == 2.0 ** -60


@pytest.mark.parametrize("n,at", [(1, 0), (1, 15), (9, 11), (16, 5), (17, 5)])
def test_a_few_tokens_of_unusual_values(n, at):
    """Calls of at most 16 tokens and just above, behind tokens that are there already."""
    c = make_cache([at + n], 16, 2, seed=3, poison=False)
    books = R.Books(c)
    x = torch.randn(n, 2, 128, generator=torch.Generator().manual_seed(n + at)) * 1e4
    x[0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 3.0])
    x[-1, 1] = math.nan   # nothing finite in this row
    k, v = x.to(torch.bfloat16).cuda(), (x * 1e-6).to(torch.bfloat16).cuda()
    c.append(0, i32([0]), i32([at]), k, v, i32([0, n]), max_new=n)
    books.append(0, 0, at, k.double().cpu().numpy(), v.double().cpu().numpy())
    assert status() == 0 and books.same(c) is None, books.same(c)


def test_rewriting_tokens_in_the_middle_keeps_their_neighbours():
    c = make_cache([50], 32, 1, seed=5, poison=False)
    books = R.Books(c)
    k, v = [(torch.randn(10, 1, 128) * 1000).to(torch.bfloat16).cuda() for _ in range(2)]
    c.append(0, i32([0]), i32([27]), k, v, i32([0, 10]), max_new=10)
    books.append(0, 0, 27, k.double().cpu().numpy(), v.double().cpu().numpy())
    assert status() == 0 and books.same(c) is None, books.same(c)


def test_append_refuses_on_the_device_and_writes_nothing():
    c = make_cache([40, 20], 16, 1, seed=6, spare_rows=1)
    k = torch.ones(8, 1, 128, dtype=torch.bfloat16, device="cuda")
    before = R.Books(c)
    for seqs, starts, cu, most in (([0], [36], [0, 8], 8),      # beyond the sequence
                                   ([7], [0], [0, 8], 8),       # no such sequence
                                   ([-1], [0], [0, 8], 8),
                                   ([0], [0], [0, 9], 9),       # more rows than there are
                                   ([0], [0], [0, 8], 4),       # more than max_new
                                   ([0], [0], [5, 2], 4),       # backwards
                                   ([2], [0], [0, 8], 8)):      # an empty sequence
        c.append(0, i32(seqs), i32(starts), k, k, i32(cu), max_new=most)
        assert status() == E_RANGE, (seqs, starts, cu)
        assert before.same(c) is None
    c.append(0, i32([0]), i32([-1]), k, k, i32([0, 8]), max_new=8)   # skipped, not refused
    assert status() == 0 and before.same(c) is None
    c.fork(i32([0]), i32([2]))
    shared = R.Books(c)
    c.append(0, i32([2]), i32([0]), k, k, i32([0, 8]), max_new=8)    # a page that two sequences hold
    assert status() == E_RANGE and shared.same(c) is None


# ---------------------------------------------------------------------------------------- books
@pytest.mark.parametrize("page,hkv,layers,seed", [(16, 1, 1, 0), (32, 3, 2, 1), (64, 8, 2, 2), (128, 2, 1, 3), (16, 2, 3, 4)])
def test_random_histories(page, hkv, layers, seed):
    """Reserve, append, fork, copy, free and compact in random order, refused calls among them, against plain Python."""
    rng = np.random.RandomState(seed)
    c = make_cache([0] * 12, page, hkv, layers=layers, extra=60, seed=seed, per_row=9, poison=False)
    books = R.Books(c)
    refused = 0
    for step in range(120):
        op = rng.choice(["reserve", "reserve", "fork", "copy", "free", "compact"])
        n = rng.randint(1, 5)
        some = rng.permutation(12)[:n].tolist() if rng.rand() < 0.9 else rng.randint(-1, 13, n).tolist()
        if op == "reserve":
            add = [int(a) for a in rng.randint(0, 2 * page, n)]
            want = books.reserve(some, add)
            starts = c.reserve(i32(some), i32(add))
            assert starts.tolist() == (want if want is not None else [-1] * n)
            ok = want is not None
            if ok and sum(add):
                k, v = [torch.from_numpy(rng.randn(sum(add), hkv, 128) * 2.0 ** rng.randint(-4, 5)).to(torch.bfloat16).cuda() for _ in range(2)]
                cu = np.concatenate([[0], np.cumsum(add)]).tolist()
                layer = int(rng.randint(layers))
                c.append(layer, i32(some), starts, k, v, i32(cu), max_new=max(add))
                for i, s in enumerate(some):
                    books.append(layer, s, want[i], k[cu[i]:cu[i + 1]].double().cpu().numpy(), v[cu[i]:cu[i + 1]].double().cpu().numpy())
        elif op in ("fork", "copy"):
            src = [int(s) for s in rng.randint(0, 12, n)]
            if rng.rand() < 0.7:
                some = [s for s in range(12) if books.lens[s] == 0][:n] or some
                src = src[:len(some)]
            ok = books.branch(src, some, op == "fork")
            getattr(c, op)(i32(src), i32(some))
        elif op == "free":
            ok = books.free(some)
            c.free(i32(some))
        else:
            books.compact()
            c.compact()
            ok = True
        st = status()
        assert (st == 0) == ok and st in (0, E_RANGE, E_NOMEM), (step, op, st, ok)
        refused += not ok
        if step % 10 == 9 or not ok:
            diff = books.same(c)
            assert diff is None, (step, op, diff)
    assert refused > 3


def test_reserve_of_many_pages_at_once():
    import magi_b200 as mb
    c = mb.TokenPagedKVCache(1, 40000, 16, 1, 600, 2500)
    c.page_refs[::7] = 1
    books = R.Books(c)
    n_new = [int(v) for v in np.random.RandomState(0).randint(0, 900, 500)]
    seqs = np.random.RandomState(1).permutation(600)[:500].tolist()
    starts = c.reserve(i32(seqs), i32(n_new))
    assert starts.tolist() == books.reserve(seqs, n_new) and books.same(c) is None and status() == 0
    c.free(i32(seqs))
    books.free(seqs)
    assert books.same(c) is None
    c.reserve(i32([0]), i32([40000]))
    books.reserve([0], [40000])
    assert books.same(c) is None and status() == 0
    c.compact()
    books.table, books.refs = [[] for _ in range(600)], None
    assert status() == 0 and int((c.page_refs[:int((c.page_refs > 0).sum())] == 0).sum()) == 0


def test_refusals_leave_everything_as_it_was():
    c = make_cache([20, 40, 0, 0], 16, 1, extra=2, seed=3, per_row=8)
    books = R.Books(c)
    for call, want in ((lambda: c.reserve(i32([0, 0]), i32([1, 1])), E_RANGE),
                       (lambda: c.reserve(i32([0, 9]), i32([1, 1])), E_RANGE),
                       (lambda: c.reserve(i32([0, -1]), i32([1, 1])), E_RANGE),
                       (lambda: c.reserve(i32([0, 1]), i32([1, -1])), E_RANGE),
                       (lambda: c.reserve(i32([0]), i32([109])), E_RANGE),          # beyond the table row
                       (lambda: c.reserve(i32([0]), i32([2 ** 31 - 1])), E_RANGE),
                       (lambda: c.reserve(i32([0, 1]), i32([1, 57])), E_NOMEM),
                       (lambda: c.fork(i32([0]), i32([1])), E_RANGE),               # not empty
                       (lambda: c.fork(i32([0, 1]), i32([2, 2])), E_RANGE),
                       (lambda: c.fork(i32([0, 2]), i32([2, 3])), E_RANGE),         # a source that this call fills
                       (lambda: c.fork(i32([2]), i32([2])), E_RANGE),
                       (lambda: c.fork(i32([4]), i32([2])), E_RANGE),
                       (lambda: c.copy(i32([1]), i32([2])), E_NOMEM),
                       (lambda: c.free(i32([0, 0])), E_RANGE),
                       (lambda: c.free(i32([0, 4])), E_RANGE)):
        r = call()
        assert status() == want
        assert r is None or (r == -1).all()
        assert books.same(c) is None
    c.free(i32([2, 3]))    # empty already: nothing to do
    assert status() == 0 and books.same(c) is None
    c.fork(i32([2]), i32([3]))   # an empty sequence has empty branches
    assert status() == 0 and books.same(c) is None
    empty = i32([])
    c.reserve(empty, empty), c.fork(empty, empty), c.copy(empty, empty), c.free(empty)
    assert status() == 0 and books.same(c) is None


# ---------------------------------------------------------------------------------------- together
def _step(mb, c, layer_in, seqs, ones, freq, pos):
    """One decode step of a toy model of two layers: rotate, reserve, append, attend."""
    starts = c.reserve(seqs, ones)
    outs = []
    for layer, (q, k, v) in enumerate(layer_in):
        c.append(layer, seqs, starts, mb.rotary(k, starts, freq), v)
        outs.append(mb.paged_attn(mb.rotary(q, starts, freq), c, layer, seqs))
    return starts, outs


def test_a_serving_loop():
    """Prompts read in, branches forked, tokens appended, a branch dropped, the pool compacted: attention of the result
    equals attention over the exact history (up to the 8-bit codes, which the reference reads from the cache)."""
    import magi_b200 as mb
    hq, hkv, layers = 12, 2, 2
    c = mb.TokenPagedKVCache(layers, 64, 16, hkv, 8, 20)
    freq, _ = mb.rotary_frequencies(96)
    books = R.Books(c)
    g = torch.Generator(device="cuda").manual_seed(0)
    n = [37, 90]
    starts = c.reserve(i32([0, 1]), i32(n))
    books.reserve([0, 1], n)
    cu = [0, 37, 127]
    pos = torch.cat([torch.arange(37), torch.arange(90)]).int().cuda()
    for layer in range(layers):
        q, k, v = [torch.randn(127, h, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv)]
        k = mb.rotary(k, pos, freq)
        c.append(layer, i32([0, 1]), starts, k, v, i32(cu), max_new=90)
        for i in range(2):
            books.append(layer, i, 0, *[t[cu[i]:cu[i + 1]].double().cpu().numpy() for t in (k, v)])
        out, _ = mb.paged_attn(mb.rotary(q, pos, freq), c, layer, i32([0, 1]), i32(cu), max_q=90)
        ref, _, tol, _ = R.attention(books, layer, mb.rotary(q, pos, freq).double().cpu().numpy(), [0, 1], cu, hkv)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()
    c.fork(i32([0, 0, 1]), i32([2, 5, 4]))
    books.branch([0, 0, 1], [2, 5, 4], True)
    assert books.same(c) is None
    live = [0, 1, 2, 4, 5]
    for step in range(20):
        if step == 9:
            c.free(i32([1, 0]))
            books.free([1, 0])
            c.compact()
            books.compact()
            live = [2, 4, 5]
            assert books.same(c) is None
        seqs, ones = i32(live), i32([1] * len(live))
        ins = [[torch.randn(len(live), h, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv)] for _ in range(layers)]
        starts, outs = _step(mb, c, ins, seqs, ones, freq, None)
        want = books.reserve(live, [1] * len(live))
        assert starts.tolist() == want
        for layer, (q, k, v) in enumerate(ins):
            kr = mb.rotary(k, starts, freq)
            for i, s in enumerate(live):
                books.append(layer, s, want[i], kr[i:i + 1].double().cpu().numpy(), v[i:i + 1].double().cpu().numpy())
        assert books.same(c) is None, step
        for layer, (q, k, v) in enumerate(ins):
            ref, _, tol, _ = R.attention(books, layer, mb.rotary(q, starts, freq).double().cpu().numpy(), live, list(range(len(live) + 1)), hkv)
            assert (np.abs(outs[layer][0].double().cpu().numpy() - ref) <= tol).all()
    assert status() == 0


def test_a_captured_step_replays():
    """The whole step in one graph, replayed over page boundaries, equals the eager steps; another graph of the same cache
    lives beside it."""
    import magi_b200 as mb
    hq, hkv, layers = 6, 1, 2
    lens = [14, 300, 0]

    def fresh():
        return make_cache(lens, 16, hkv, layers=layers, extra=12, seed=4, per_row=24)

    freq, _ = mb.rotary_frequencies(128)
    g = torch.Generator(device="cuda").manual_seed(1)
    steps = [[[torch.randn(3, h, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv)] for _ in range(layers)] for _ in range(8)]
    seqs, ones = i32([0, 1, 2]), i32([1, 1, 1])
    eager, want = fresh(), []
    for ins in steps:
        want.append([o[0].clone() for o in _step(mb, eager, ins, seqs, ones, freq, None)[1]])
    c = fresh()
    saved = [t.clone() for t in (c.page_table, c.seq_lens, c.page_refs)]
    static = [[t.clone() for t in layer] for layer in steps[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(mb, c, static, seqs, ones, freq, None)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, outs = _step(mb, c, static, seqs, ones, freq, None)
    with torch.cuda.graph(other):
        look = mb.paged_attn(static[0][0], c, 0, seqs)
    c2 = fresh()
    for t, s in zip((c.k8, c.v8, c.k_scale, c.v_scale), (c2.k8, c2.v8, c2.k_scale, c2.v_scale)):
        t.view(torch.uint8).copy_(s.view(torch.uint8))
    for t, s in zip((c.page_table, c.seq_lens, c.page_refs), saved):
        t.copy_(s)
    for ins, w in zip(steps, want):
        for a, b in zip(static, ins):
            for x, y in zip(a, b):
                x.copy_(y)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, w):
            assert torch.equal(o[0], e)
        assert torch.equal(look[0], mb.paged_attn(static[0][0], c, 0, seqs)[0])
    assert status() == 0
    assert R.Books(eager).same(c) is None


# ---------------------------------------------------------------------------------------- arguments
def test_arguments_are_checked():
    import magi_b200 as mb
    c = make_cache([10], 16, 2, seed=1)
    q, k = strided_bf16(1, 4, 1), strided_bf16(1, 2, 2)
    one, seqs = i32([1]), i32([0])
    for bad in (lambda: mb.TokenPagedKVCache(1, 4, 48, 1, 1, 1), lambda: mb.TokenPagedKVCache(0, 4, 16, 1, 1, 1),
                lambda: c.reserve(torch.tensor([0]), one), lambda: c.reserve(seqs.long(), one), lambda: c.reserve(seqs, i32([1, 2])),
                lambda: c.reserve(i32([[0]]), one), lambda: c.reserve(i32([0, 0, 0])[::2], i32([1, 1])), lambda: c.reserve(i32([0] * 1025), i32([0] * 1025)),
                lambda: c.append(0, seqs, one, k.float(), k), lambda: c.append(0, seqs, one, k[:, :1], k[:, :1]),
                lambda: c.append(0, seqs, one, k, k[:0]), lambda: c.append(0, seqs, one, k[:0], k[:0]),
                lambda: c.append(0, seqs, one, k, k, i32([0])), lambda: c.append(0, seqs, one, k, k, max_new=2),
                lambda: mb.paged_attn(q.cpu(), c, 0, seqs), lambda: mb.paged_attn(q.half(), c, 0, seqs),
                lambda: mb.paged_attn(q[:, :3], c, 0, seqs), lambda: mb.paged_attn(q, c, 0, i32([0, 0])),
                lambda: mb.paged_attn(q, c, 0, seqs, window=-1), lambda: mb.paged_attn(q, c, 0, seqs, i32([0, 1, 1])),
                lambda: mb.paged_attn(q, c, 0, seqs, out=q[:0]), lambda: mb.paged_attn(q, c, 0, seqs, max_q=2)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: mb.paged_attn(q, c, 1, seqs), lambda: mb.paged_attn(q, c, -1, seqs), lambda: c.append(1, seqs, one, k, k),
                lambda: mb.paged_attn(torch.zeros(1, 4, 132, dtype=torch.bfloat16, device="cuda")[..., 2:130], c, 0, seqs)):
        with pytest.raises(mb.MagiError):
            bad()
    assert mb.paged_attn(q[:0], c, 0, i32([]))[0].shape == (0, 4, 128)
    assert status() == 0


def test_a_long_tail_behind_one_large_weight():
    """One key takes about half of the softmax, 60000 others share the rest: their weights, 2^-16 of the largest, must not
    be rounded away.  Values: 0 at the large key, 1 elsewhere."""
    import magi_b200 as mb
    n = 60001
    c = make_cache([n], 128, 1, seed=30, poison=False)
    ids = c.page_table[0].long()
    c.k8.view(torch.uint8).zero_()
    c.v8.view(torch.uint8).fill_(0x38)          # 1.0
    c.k_scale.fill_(1.0), c.v_scale.fill_(1.0)
    q = torch.zeros(1, 6, 128, dtype=torch.bfloat16, device="cuda")
    q[0, :, 0] = 12.0
    for where in (0, 5000, n - 1):
        c.k8.view(torch.uint8).zero_()
        c.v8.view(torch.uint8).fill_(0x38)
        page, off = int(ids[where // 128]), where % 128
        c.k8.view(torch.uint8)[0, page, 0, off, 0] = 0x52   # 10.0: the score 12 * 10 / sqrt(128) = 10.607 nats = 15.3 bits
        c.v8.view(torch.uint8)[0, page, 0, off] = 0
        out, lse = mb.paged_attn(q, c, 0, i32([0]))
        big = math.exp(12 * 10 / math.sqrt(128))
        want = (n - 1) / (n - 1 + big)
        # every small weight is the same number and rounds the same way, by at most 2^-3 of it (e5m2): the bound of the result
        assert abs(float(out.double().mean()) - want) <= (2.0 ** -8 + 2.0 ** -3) * want
        assert abs(float(lse[0, 0]) - math.log(n - 1 + big)) <= 1e-4


def test_a_scale_that_is_no_positive_number_is_refused():
    import magi_b200 as mb
    c = make_cache([10], 16, 2, seed=1)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            mb.paged_attn(strided_bf16(1, 4, 1), c, 0, i32([0]), softmax_scale=scale)


def test_numbers_beyond_32_bits_do_not_wrap():
    import magi_b200 as mb
    c = make_cache([10], 16, 2, seed=1)
    q, k = strided_bf16(1, 4, 1), strided_bf16(1, 2, 2)
    for bad in (lambda: mb.paged_attn(q, c, 2 ** 32, i32([0])), lambda: c.append(-2 ** 32, i32([0]), i32([9]), k, k)):
        with pytest.raises(mb.MagiError):
            bad()
    with pytest.raises(ValueError):
        c.append(0, i32([0]), i32([9]), k, k, i32([0, 1]), max_new=2 ** 32 + 1)
    with pytest.raises(ValueError):
        mb.paged_attn(q, c, 0, i32([0]), i32([0, 1]), max_q=2 ** 32 + 1)


# ---------------------------------------------------------------------------------------- prompts of short and full units
def spread_scales(c, seed, lo=-12, hi=4):
    """Scales of V that differ from page to page by far more than the codes do."""
    g = torch.Generator().manual_seed(seed)
    c.v_scale.copy_(2.0 ** torch.randint(lo, hi + 1, c.v_scale.shape, generator=g).float())


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("short,full", [(10, 40), (21, 22), (6, 43)])
def test_short_units_of_many_tiles_in_front_of_full_ones(page, short, full):
    """A short unit (up to 128 rows) leaves the second row tile out for dozens of tiles; then comes a unit of 129 to 256 rows."""
    pairs = 150
    c = make_cache([3001, 611], page, 1, seed=page + short, poison=False)
    spread_scales(c, short)
    n_q = [short, full] * pairs
    cu = np.concatenate([[0], np.cumsum(n_q)]).tolist()
    check_attn(c, strided_bf16(cu[-1], 6, 37), [0, 1] * pairs, cu)


@pytest.mark.parametrize("window", [0, 4000])
def test_full_units_over_many_tiles(window):
    """Units of two row tiles over 9001 keys, each split over several blocks, behind remainders of up to 128 rows."""
    c = make_cache([9001, 9000, 5003], 32, 2, seed=41, poison=False)
    spread_scales(c, 3, -8, -4)
    n_q = [100, 131, 43]
    check_attn(c, strided_bf16(sum(n_q), 12, 43), [0, 1, 2], np.concatenate([[0], np.cumsum(n_q)]).tolist(), window=window)


# ---------------------------------------------------------------------------------------- one large weight and many small ones
# What the kernel's own roundings may do to a row with weights p relative to the row's largest (times its page's scale of V):
# three e5m2 terms of its fp16 value leave 2^-10 of a weight at most, beside 2^-11 of the rounding to fp16, and e5m2's smallest
# step of 2^-16 is off by 2^-17 of a reference of 2^12 at least: 2^-29.  The queries' two terms change a score by ds (see paged_ref.attention), a weight by 2 ds of
# it; the fp32 exponent and sums by 2^-14; the result is rounded to bf16, 2^-8 of it.
def flat_cache(n, seed):
    """A sequence of n keys that are zero, values one."""
    c = make_cache([n], 128, 1, seed=seed, poison=False)
    c.k8.view(torch.uint8).zero_()
    c.v8.view(torch.uint8).fill_(0x38)          # 1.0
    c.k_scale.fill_(1.0), c.v_scale.fill_(1.0)
    return c


@pytest.mark.parametrize("n,n_q,entries", [(8191, 1, 600), (131072, 1, 128), (8191, 4, 600), (8191, 40, 150), (40000, 40, 40)])
def test_small_weights_keep_their_bits(n, n_q, entries):
    import magi_b200 as mb
    # `entries` entries that all are the same rows of one sequence, so that a block's part of the work is a whole unit or hundreds
    # of tiles of it: key `where` has the largest score and no values, the others `level` nats less each
    c = flat_cache(n, n_q)
    ids = c.page_table[0].long()
    for level in (7.0, 9.5, 10.6, 12.0, 13.3, 14.7):
        for where in (0, n // 2, n - n_q):
            page, off = int(ids[where // 128]), where % 128
            c.k8.view(torch.uint8).zero_()
            c.v8.view(torch.uint8).fill_(0x38)
            c.k8.view(torch.uint8)[0, page, 0, off, 0] = 0x48      # 4.0
            c.v8.view(torch.uint8)[0, page, 0, off] = 0
            q = torch.zeros(n_q, 6, 128, dtype=torch.bfloat16, device="cuda")
            q[:, :, 0] = level * math.sqrt(128) / 4
            out, lse = mb.paged_attn(q.repeat(entries, 1, 1), c, 0, i32([0] * entries), i32((np.arange(entries + 1) * n_q).tolist()), max_q=n_q)
            score = float(q[0, 0, 0]) * 4 / math.sqrt(128)
            seen = n - n_q + np.arange(n_q)[:, None] + 0.0      # small ones: all keys up to the row's but the large one
            total = seen * math.exp(-score) + 1
            want = seen * math.exp(-score) / total
            tol = (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -14) * want + 2.0 ** -29 * seen / total
            err = np.abs(out.double().cpu().numpy().reshape(entries, n_q, -1) - want)
            assert (err <= tol).all(), (level, where, float((err / want).max()))
            assert (np.abs(lse.double().cpu().numpy().reshape(entries, n_q, 6) - (score + np.log(total))[None]) <= 2.0 ** -16 + 2.0 ** -20 * score).all()
    assert status() == 0


@pytest.mark.parametrize("n,n_q,entries", [(8191, 1, 600), (60001, 1, 128), (8191, 4, 600), (8191, 40, 150)])
@pytest.mark.parametrize("mass", [0.55, 0.95])
def test_a_key_that_holds_most_of_the_mass(n, n_q, entries, mass):
    """Random scores and values; the large key's own values are small, so that the result is what the small weights bring.  The
    roundings of the weights are independent: they move a row by sqrt(sum (dp v)^2), 2^-9.4 sqrt(sum (p v)^2) at most, which is
    2^-9.4 of the row's own size up to the spread of such sums (taken as a factor of 2), beside bf16's 2^-8; 2^-29 of the
    reference over n keys adds 2^-29 sqrt(n) to sqrt(sum p^2) >= (1 - mass) / sqrt(n).  The queries' entries are at most 2.5 and
    sum |k| below 120, so a score is off by ds <= 2^-17 * 2.5 * 120 / sqrt(128) = 2^-12.3, a weight by 2^-11.3 of it."""
    import magi_b200 as mb
    c = make_cache([n], 64, 1, seed=n_q, poison=False)
    ids = c.page_table[0].long()
    c.k_scale.fill_(2.0 ** -7), c.v_scale.fill_(2.0 ** -7)
    c.k8.view(torch.uint8)[0, :, 0, :, 0] = 0
    page, off = int(ids[0]), 5
    c.k8.view(torch.uint8)[0, page, 0] = 0                  # the others of its page: scores of zero
    c.k8.view(torch.uint8)[0, page, 0, off, 0] = 0x7c       # 384
    c.k_scale[0, page, 0] = 1.0
    c.v8.view(torch.uint8)[0, page, 0, off] = 0
    q = (torch.randn(n_q, 6, 128, generator=torch.Generator().manual_seed(5)) * 0.5).to(torch.bfloat16).cuda()
    others = R.attention(R.Books(c), 0, q.double().cpu().numpy() * (np.arange(128) > 0), [0], [0, n_q], 1)[1]
    q[:, :, 0] = torch.from_numpy((others + math.log(mass / (1 - mass))) * math.sqrt(128) / 384).to(torch.bfloat16).cuda()
    ref, ref_l, _, tol_l = R.attention(R.Books(c), 0, q.double().cpu().numpy(), [0], [0, n_q], 1)
    out, lse = mb.paged_attn(q.repeat(entries, 1, 1), c, 0, i32([0] * entries), i32((np.arange(entries + 1) * n_q).tolist()), max_q=n_q)
    o = out.double().cpu().numpy().reshape(entries, n_q, 6, 128)
    rel = np.sqrt(((o - ref) ** 2).sum(-1) / (ref ** 2).sum(-1))
    assert (rel <= 2.0 ** -8 + 2 * (2.0 ** -9.4 + 2.0 ** -11.3 + 2.0 ** -29 * n / (1 - mass))).all(), float(rel.max())
    assert float(q.abs().max()) <= 2.5 and (np.abs(lse.double().cpu().numpy().reshape(entries, n_q, 6) - ref_l) <= tol_l).all() and status() == 0


# ---------------------------------------------------------------------------------------- reservations appended in parts
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("parts", [[(0, 24), (24, 32)], [(0, 1), (1, 2), (2, 200)], [(100, 180), (0, 100)], [(17, 40), (60, 75), (0, 17), (40, 60), (75, 80)]])
def test_a_reservation_appended_in_parts(page, parts):
    """Pages whose last owner left scales of 2^40 behind take the scale of what is appended now, in any order of the parts, and
    layer by layer."""
    import magi_b200 as mb
    hkv, layers, total = 2, 2, max(b for _, b in parts)
    c = mb.TokenPagedKVCache(layers, 40, page, hkv, 4, 20)
    big = torch.full((300, hkv, 128), 2.0 ** 40, device="cuda").to(torch.bfloat16)
    c.reserve(i32([3]), i32([300]))
    for layer in range(layers):
        c.append(layer, i32([3]), i32([0]), big, big, i32([0, 300]), max_new=300)
    c.free(i32([3]))
    start = 5
    assert c.reserve(i32([1]), i32([start])).tolist() == [0]
    g = torch.Generator().manual_seed(page)
    k, v = [(torch.randn(start + total, hkv, 128, generator=g) * torch.exp(torch.randn(start + total, 1, 1, generator=g))).to(torch.bfloat16).cuda() for _ in range(2)]
    for layer in range(layers):
        c.append(layer, i32([1]), i32([0]), k[:start], v[:start], i32([0, start]), max_new=start)
    assert c.reserve(i32([1]), i32([total])).tolist() == [start]
    for layer in range(layers):
        books = R.Books(c)
        for s in (books.ks, books.vs):
            s[layer, books.table[1][1 if start % page else 0:]] = 2.0 ** -60   # pages that nothing has been written to
        for a, b in parts:
            c.append(layer, i32([1]), i32([start + a]), k[start + a:start + b], v[start + a:start + b], i32([0, b - a]), max_new=b - a)
            books.append(layer, 1, start + a, *[t[start + a:start + b].double().cpu().numpy() for t in (k, v)])
        got = R.Books(c)
        for name in ("k8", "v8", "ks", "vs"):
            for slot, p in enumerate(books.table[1]):
                held = min(start + total - slot * page, page)
                a, b = getattr(books, name)[layer, p], getattr(got, name)[layer, p]
                if name[1] == "8":
                    a, b = a[:, :held], b[:, :held]
                assert np.array_equal(a, b), (layer, name, slot)
        for h in range(hkv):
            gk, gv = got.kv(layer, 1, h)
            for x, y in ((gk, k), (gv, v)):
                y = y[:, h].double().cpu().numpy()
                # a code is off by 2^-4 of its value, or 2^-10 of the page's scale, each time it is rounded (part by part)
                top = np.concatenate([np.full((min(page, len(y) - at), 1), np.abs(y[at:at + page]).max()) for at in range(0, len(y), page)])
                assert (np.abs(x - y) <= 2.0 ** -4 * np.abs(y) * (1 + 2.0 ** -3) + len(parts) * 2.0 ** -10 * top * 2 / 224).all()
    assert status() == 0


@pytest.mark.parametrize("how", ["fork", "copy", "compact"])
def test_pages_that_move_before_they_are_written(how):
    """A page that is reserved, not yet written, and then copied or moved takes no scale from its past either."""
    import magi_b200 as mb
    page = 32
    c = mb.TokenPagedKVCache(1, 12, page, 1, 4, 6)
    big = torch.full((12 * page, 1, 128), 2.0 ** 40, device="cuda").to(torch.bfloat16)
    c.reserve(i32([3, 2]), i32([6 * page, 6 * page]))
    c.append(0, i32([3, 2]), i32([0, 0]), big, big, i32([0, 6 * page, 12 * page]), max_new=6 * page)
    c.free(i32([3, 2]))
    if how == "compact":
        c.reserve(i32([3]), i32([2 * page]))   # in front, and gone before the move
    x = torch.randn(page + 20, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    c.reserve(i32([0]), i32([page + 20]))
    c.append(0, i32([0]), i32([0]), x[:page], x[:page], i32([0, page]), max_new=page)   # its first page only
    row = 0
    if how == "compact":
        c.free(i32([3]))
        c.compact()
    else:
        getattr(c, how)(i32([0]), i32([1]))
        row = 1
    for a, b in ((page, page + 8), (page + 8, page + 20)):
        c.append(0, i32([row]), i32([a]), x[a:b], x[a:b], i32([0, b - a]), max_new=b - a)
    assert status() == 0
    got = R.Books(c)
    k, v = got.kv(0, row, 0)
    want = x[:, 0].double().cpu().numpy()
    for t in (k, v):   # the scale is at most 2^-6 (values below 7): codes are off by 2^-4 of a value or half a step, 2^-10, of it
        assert (np.abs(t - want) <= 2.0 ** -4 * np.abs(want) + 2 * 2.0 ** -16).all()


def test_two_reservations_appended_the_later_one_first():
    import magi_b200 as mb
    c = mb.TokenPagedKVCache(2, 2, 32, 1, 2, 2)
    big = torch.full((64, 1, 128), 2.0 ** 40, device="cuda").to(torch.bfloat16)
    c.reserve(i32([1]), i32([64]))
    for layer in range(2):
        c.append(layer, i32([1]), i32([0]), big, big, i32([0, 64]), max_new=64)
    c.free(i32([1]))
    x = torch.randn(30, 1, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    c.reserve(i32([0]), i32([20]))
    c.reserve(i32([0]), i32([10]))
    for layer, parts in enumerate((((20, 30), (0, 20)), ((0, 20), (20, 30)))):   # the second layer in order: the page is continued by then
        for a, b in parts:
            c.append(layer, i32([0]), i32([a]), x[a:b], x[a:b], i32([0, b - a]), max_new=b - a)
        for t in R.Books(c).kv(layer, 0, 0):
            want = x[:, 0].double().cpu().numpy()
            assert (np.abs(t - want) <= 2.0 ** -4 * np.abs(want) + 2 * 2.0 ** -16).all()
    assert status() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 120])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,n_q,n", [(6, 2, 0), (6, 2, 200), (6, 5, 1), (6, 5, 131), (6, 60, 20), (6, 300, 200), (6, 300, 300), (6, 129, 700)])
def test_the_largest_windows_are_none(window, causal, hq, n_q, n):
    """With more rows than keys, too, so that positions are negative; in every form."""
    import magi_b200 as mb
    c = make_cache([n], 64, 1, seed=n + n_q)
    q = strided_bf16(n_q, hq, 47)
    wide = check_attn(c, q, [0], [0, n_q], window=window, causal=causal)
    assert np.array_equal(wide, check_attn(c, q, [0], [0, n_q], causal=causal))


def test_a_scale_that_32_bits_do_not_hold_is_refused():
    import magi_b200 as mb
    c = make_cache([300], 16, 1, seed=1)
    q = strided_bf16(1, 6, 1)
    for scale in (1e-46, 1e-300, 3.1e38, 1e39, 1e300):
        with pytest.raises(ValueError):
            mb.paged_attn(q, c, 0, i32([0]), softmax_scale=scale)
    # the smallest that it holds: every key weighs the same
    check_attn(c, q, [0], [0, 1], softmax_scale=2.0 ** -149)
    check_attn(c, q, [0], [0, 1], softmax_scale=2.0 ** -126)


def test_results_that_share_memory_with_the_queries():
    """out may be q itself, or lie apart from it, between q's own heads too; anything else is refused."""
    import magi_b200 as mb
    c = make_cache([300, 5000, 77], 64, 2, seed=3)
    for n_q in (1, 8, 70):
        cu = [0, n_q, 2 * n_q, 3 * n_q]
        args = (c, 0, i32([0, 1, 2]), i32(cu), n_q)
        packed = strided_bf16(3 * n_q + 1, 8, 51).contiguous()
        q = packed[:-1, :4]
        want, _ = mb.paged_attn(q, *args)
        beside, rest = packed.clone(), packed.clone()
        got, _ = mb.paged_attn(beside[:-1, :4], *args, out=beside[:-1, 4:])
        rest[:-1, 4:] = want
        assert torch.equal(got, want) and torch.equal(beside, rest)
        for bad in (packed[1:, :4], packed[:-1, 1:5], packed[:-1, 3:7], packed.view(-1, 16, 64)[:-1, ::2].as_strided((3 * n_q, 4, 128), (1024, 256, 1))):
            with pytest.raises(ValueError):
                mb.paged_attn(q, *args, out=bad)
        again, _ = mb.paged_attn(q, *args, out=q)
        assert again is q and torch.equal(q, want)
    assert status() == 0


def test_rows_beyond_32_bits_do_not_wrap():
    import magi_b200 as mb
    c = make_cache([10], 16, 1, seed=1)
    before = R.Books(c)
    k = torch.zeros(1, 1, 128, dtype=torch.bfloat16, device="cuda").expand(2 ** 32 + 1, 1, 128)
    with pytest.raises(ValueError, match="32-bit"):
        c.append(0, i32([0]), i32([9]), k, k, i32([0, 1]), max_new=1)
    with pytest.raises(ValueError, match="32-bit"):
        mb.paged_attn(k, c, 0, i32([0]), i32([0, 1]), max_q=1, out=torch.empty(1, 1, 128, dtype=torch.bfloat16, device="cuda"))
    assert status() == 0 and before.same(c) is None


def test_a_second_row_tile_that_waits_longer_than_a_wait_may_last():
    """Every block has short units for about a second; the full unit behind them finds its second row tile still there."""
    import magi_b200 as mb
    n, entries, n_q = 6_000_000, 1000, 21
    pages = -(-n // 128)
    c = mb.TokenPagedKVCache(1, pages + 6, 128, 1, 2, pages)
    g = torch.Generator(device="cuda").manual_seed(3)
    for t in (c.k8, c.v8):
        for part in t.view(-1, 128).split(1 << 20):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") * 60)
    c.k_scale.fill_(2.0 ** -6), c.v_scale.fill_(2.0 ** -6)
    assert c.reserve(i32([0, 1]), i32([n, 700])).tolist() == [0, 0]
    cu = [n_q * i for i in range(entries + 1)] + [n_q * entries + 43]
    q = strided_bf16(n_q, 6, 53).repeat(entries, 1, 1)
    q = torch.cat([q, strided_bf16(43, 6, 54)])
    args = (c, 0, i32([0] * entries + [1]), i32(cu))
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out, lse = mb.paged_attn(q, *args, max_q=43)
    end.record()
    torch.cuda.synchronize()
    assert status() == 0
    assert start.elapsed_time(end) > 600, "too little work to show it"
    for rows in (out[:-43].view(entries, n_q, 6, 128), lse[:-43].view(entries, n_q, 6)):
        assert rows.isfinite().all()
    assert float((lse[:-43].view(entries, n_q, 6) - lse[:n_q]).abs().max()) <= 2.0 ** -15 + 2.0 ** -19 * 20   # the same rows, in other parts
    ids = c.page_table[1, :6].long()
    k, v = [(t[0, ids, 0].double() * s[0, ids, 0].double()[:, None, None]).reshape(-1, 128)[:700] for t, s in ((c.k8, c.k_scale), (c.v8, c.v_scale))]
    score = torch.einsum("thd,kd->thk", q[-43:].double(), k) / math.sqrt(128)
    seen = torch.arange(700, device="cuda")[None, None] <= 657 + torch.arange(43, device="cuda")[:, None, None]
    p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
    want, size = p @ v, p @ v.abs()
    # queries below 4.5, sum |k| below 130: ds <= 2^-17 * 4.5 * 130 / sqrt(128); 2^-9.4 of a weight, 2 ds, 2^-14: below 2^-8 in all
    assert float(q.abs().max()) < 4.5 and float(k.abs().sum(1).max()) < 130
    assert ((out[-43:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * size).all()


# ---------------------------------------------------------------------------------------- far pages, streams, rewinding
def test_pages_beyond_32_bits():
    """A pool of 5 GB each for K and V in two layers, the pages in use at its far end."""
    import magi_b200 as mb
    page, hkv, n_pages = 128, 2, 82000
    c = mb.TokenPagedKVCache(2, n_pages, page, hkv, 4, 40)
    assert c.k8.numel() > 2 ** 32 + 2 ** 29
    c.page_refs[:n_pages - 20] = 1
    rng = np.random.RandomState(0)
    n = [300, 1, 129]
    starts = c.reserve(i32([0, 1, 2]), i32(n))
    assert starts.tolist() == [0, 0, 0]
    cu = [0, 300, 301, 430]
    k, v = [torch.from_numpy(rng.randn(430, hkv, 128)).to(torch.bfloat16).cuda() for _ in range(2)]
    for layer in (1, 0):
        c.append(layer, i32([0, 1, 2]), starts, k * (layer + 1), v, i32(cu), max_new=300)
    c.copy(i32([0]), i32([3]))

    def check(rows):
        q = strided_bf16(len(rows), 6, 61)
        for layer in range(2):
            out, lse = mb.paged_attn(q, c, layer, i32(rows))
            for i, s in enumerate(rows):
                ids = c.page_table[s, :-(-int(c.seq_lens[s]) // page)].long()
                at = (0, 1, 2, 0)[s]
                for h in range(hkv):
                    kk, vv = [(t[layer, ids, h].double() * z[layer, ids, h].double()[:, None, None]).reshape(-1, 128)[:n[at]] for t, z in ((c.k8, c.k_scale), (c.v8, c.v_scale))]
                    # what was appended, to within a code's half step
                    want = (k * (layer + 1))[cu[at]:cu[at + 1], h].double()
                    assert ((kk - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * 2.0 ** -5).all()
                    p = torch.softmax(q[i, h * 3:h * 3 + 3].double() @ kk.T / math.sqrt(128), 1)
                    assert ((out[i, h * 3:h * 3 + 3].double() - p @ vv).abs() <= 2.0 ** -8 * (p @ vv).abs() + 2.0 ** -8 * (p @ vv.abs())).all()

    check([0, 1, 2, 3])
    c.free(i32([0]))
    c.page_refs[:n_pages - 20] = 0
    c.compact()
    assert int(c.page_refs.sum()) == int((c.page_refs[:6] > 0).sum()) == 6
    check([3, 1, 2])
    assert status() == 0


def test_layers_on_streams_of_their_own():
    """Appends and attention of different layers at once, over pages whose last owner's scales were large."""
    import magi_b200 as mb
    layers, hkv, n = 4, 2, [700, 33, 1500]
    cu, total = [0, 700, 733, 2233], 2233

    def fresh():
        c = mb.TokenPagedKVCache(layers, 200, 16, hkv, 4, 120)
        big = torch.full((1900, hkv, 128), 2.0 ** 30, device="cuda").to(torch.bfloat16)
        c.reserve(i32([3]), i32([1900]))
        for layer in range(layers):
            c.append(layer, i32([3]), i32([0]), big, big, i32([0, 1900]), max_new=1900)
        c.free(i32([3]))
        return c

    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = [[torch.randn(total, hkv, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(layers)] for _ in range(2)]
    q = [torch.randn(total, 6, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(layers)]
    seqs, cus = i32([0, 1, 2]), i32(cu)
    halves = []   # every entry in two parts
    for j in range(2):
        rows = [torch.arange(cu[i] + (0 if j == 0 else n[i] // 3), cu[i] + (n[i] // 3 if j == 0 else n[i])) for i in range(3)]
        halves.append((torch.cat(rows).cuda(), i32(np.concatenate([[0], np.cumsum([len(r) for r in rows])]).tolist()), i32([0 if j == 0 else x // 3 for x in n]), max(len(r) for r in rows)))

    def step(c, layer, stream):
        for (_, cu_part, first, most), kk, vv in zip(halves, ks[layer], vs[layer]):
            c.append(layer, seqs, first, kk, vv, cu_part, max_new=most, stream=stream)
        return mb.paged_attn(q[layer], c, layer, seqs, cus, max_q=1500, stream=stream)

    ks = [[x[at].contiguous() for at, _, _, _ in halves] for x in k]
    vs = [[x[at].contiguous() for at, _, _, _ in halves] for x in v]
    one = fresh()
    one.reserve(seqs, i32(n))
    want = [step(one, layer, None) for layer in range(layers)]
    books = R.Books(one)
    assert float(one.k_scale[:, one.page_table[:3][one.page_table[:3] >= 0].long()].max()) <= 2.0 ** -5
    for _ in range(5):
        c = fresh()
        c.reserve(seqs, i32(n))
        streams = [torch.cuda.Stream() for _ in range(layers)]
        torch.cuda.synchronize()
        got = [step(c, layer, streams[layer]) for layer in range(layers)]
        torch.cuda.synchronize()
        assert books.same(c) is None, books.same(c)
        for (a, la), (b, lb) in zip(want, got):
            assert torch.equal(a, b) and torch.equal(la, lb)
    assert status() == 0


def test_proposed_tokens_are_taken_back():
    """The books put back: what was proposed is gone, pages that it took are empty again, a page that goes on keeps its scale."""
    import magi_b200 as mb
    page, hkv = 16, 1
    c = mb.TokenPagedKVCache(1, 12, page, hkv, 2, 5)
    books = R.Books(c)
    rng = np.random.RandomState(1)

    def tokens(m, size):
        return [torch.from_numpy(rng.randn(m, hkv, 128) * size).to(torch.bfloat16).cuda() for _ in range(2)]

    def add(m, size):
        k, v = tokens(m, size)
        start = books.reserve([0], [m])
        assert c.reserve(i32([0]), i32([m])).tolist() == start
        c.append(0, i32([0]), i32(start), k, v, i32([0, m]), max_new=m)
        books.append(0, 0, start[0], k.double().cpu().numpy(), v.double().cpu().numpy())

    add(13, 1.0)
    for turn in range(4):
        saved = [t.clone() for t in (c.page_table, c.seq_lens, c.page_refs)]
        kept = [list(x) for x in books.table], list(books.lens), list(books.refs)
        add(7, 2.0 ** (10 * turn))   # over the page's end: the new page takes a large scale
        assert books.same(c) is None
        for t, x in zip((c.page_table, c.seq_lens, c.page_refs), saved):
            t.copy_(x)
        books.table, books.lens, books.refs = [list(x) for x in kept[0]], list(kept[1]), list(kept[2])
        add(7, 1.0)
        assert books.same(c) is None, books.same(c)
        # A weight is off by 2^-17 where it is small, the reference is 2^12 for the largest product of a weight and its page's scale
        # of V: 2^-29 of that product, times a key's codes.  It matters here, as the page that goes on keeps a scale 2^30 too large.
        q = strided_bf16(3, 4, turn)
        out, lse = mb.paged_attn(q, c, 0, i32([0]), i32([0, 3]), max_q=3)
        ref, ref_l, tol, tol_l = R.attention(books, 0, q.double().cpu().numpy(), [0], [0, 3], 1)
        key, _ = books.kv(0, 0, 0)
        n = books.lens[0]
        sv = np.repeat(books.vs[0, books.table[0], 0], page)[:n]
        codes = np.concatenate([R.CODES[books.v8[0, p, 0]] for p in books.table[0]])[:n]
        for t in range(3):
            seen = slice(0, n - 2 + t)
            w = np.exp(q[t].double().cpu().numpy() @ key[seen].T / math.sqrt(128) - ref_l[t][:, None])
            tol[t] += 2.0 ** -29 * (w * sv[seen]).max(1, keepdims=True) * np.abs(codes[seen]).sum(0)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all() and (np.abs(lse.double().cpu().numpy() - ref_l) <= tol_l).all()
    assert status() == 0
