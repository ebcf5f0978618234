"""B200: grouped-query caches (K and V per head, paged) and the attention that reads them, against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import cautreo_b200 as ct
import gqa_util as G
from gpu_util import stream

pytestmark = pytest.mark.gpu

BF16, INT8, E4M3 = ct.CT_KV_BF16, ct.CT_KV_INT8, ct.CT_KV_E4M3
MOD, BLK = ct.CT_GQA_MODULO, ct.CT_GQA_BLOCKED


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def decode(lens, heads, group, dim, page, dtype, order=MOD, window=0, seed=1, holes=(), q_extra=0, scale=0.0, poison=True,
           lens_given=None, check=True):
    g = gen(seed)
    table, n_pages = G.make_table(lens, page, g, window, holes=holes)
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    tb = table.cpu().numpy()
    if poison:                                        # slots behind a sequence's end, pages of nobody
        for s, n in enumerate(lens):
            if n % page and tb[s, n // page] >= 0:
                (pool if dtype == BF16 else scales)[int(tb[s, n // page]), :, :, n % page:] = float("nan")
        free = sorted(set(range(n_pages)) - set(tb[tb >= 0].tolist()))
        (pool if dtype == BF16 else scales)[free] = float("nan")
    hq = heads * group
    q = torch.randn(len(lens), hq * dim + q_extra, generator=g, device="cuda").bfloat16()
    qv = q[:, :hq * dim]
    lens_dev = torch.tensor(lens if lens_given is None else lens_given, dtype=torch.int32, device="cuda")
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, table.shape[1])
    plan = ct.GqaPlan(layout, len(lens), hq, window_tokens=window, head_order=order, scale=scale)
    out = torch.full((len(lens), hq, dim), 7.0, device="cuda").bfloat16()
    lse = torch.full((len(lens), hq), 7.0, device="cuda")
    for _ in range(2):                                # the second call finds the counters as the first left them
        plan.decode(qv, pool, scales, table, lens_dev, out, lse, q_stride=q.shape[1], stream=stream())
    torch.cuda.synchronize()
    if check:
        ref = G.attend(qv.reshape(len(lens), hq, dim), pool, scales, table, lens, dtype, hq, order, window,
                       scale=scale or None)
        G.check_attention(out, lse, ref, dim, max(max(lens), 1), dtype)
    return out, lse, plan


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_decode_types_and_head_sizes(dim, dtype):
    decode([1, 65, 300, 0, 17], 2, 3, dim, 64, dtype, seed=dim + dtype)


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("group,heads,order", [(1, 5, MOD), (2, 1, BLK), (8, 2, MOD), (16, 2, BLK), (17, 1, MOD), (71, 1, BLK),
                                               (40, 2, MOD)])
def test_decode_groups(group, heads, order, dtype):
    decode([33, 130, 7], heads, group, 64, 32, dtype, order=order, seed=group)


@pytest.mark.parametrize("page", [16, 48, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, INT8])
def test_decode_lengths_around_pages_and_steps(page, dtype):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 255, 257, 500, 513]
    decode(lens, 1, 4, 128, page, dtype, seed=page)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("window", [1, 15, 16, 100, 257])
def test_decode_window(window, dtype):
    decode([0, 1, 16, 99, 100, 101, 700, 333], 2, 2, 64, 32, dtype, window=window, seed=window)


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_decode_skips_unmapped_pages_and_empty_rows(dtype):
    holes = {(0, 0), (0, 3), (1, 0), (2, 1), (2, 2), (2, 3)}
    out, lse, _ = decode([300, 40, 256, 0], 2, 4, 128, 64, dtype, holes=holes, seed=5)
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all()          # every page of the row is gone
    assert (out[3] == 0).all() and torch.isinf(lse[3]).all()


@pytest.mark.parametrize("dtype,page,dim", [(BF16, 64, 128), (INT8, 16, 64), (E4M3, 128, 128)])
def test_decode_split_over_the_length(dtype, page, dim):
    _, _, plan = decode([40001], 2, 4, dim, page, dtype, seed=9)
    assert plan.workers > 100
    decode([3000, 20, 9001, 0, 4097], 1, 7, dim, page, dtype, seed=10)


def test_decode_many_short_sequences():
    lens = [(i * 37) % 90 for i in range(700)]
    decode(lens, 2, 1, 64, 16, BF16, seed=11)
    decode(lens[:300], 1, 2, 128, 16, INT8, seed=12)


def test_decode_lengths_outside_the_table_are_clamped():
    out, lse, _ = decode([128, 0], 1, 2, 64, 64, BF16, lens_given=[100000, -3], seed=13)
    assert torch.isfinite(lse[0]).all() and (out[1] == 0).all()


def test_decode_strided_queries_and_scale():
    decode([70, 200], 4, 2, 96, 16, BF16, order=BLK, q_extra=2 * 4 * 96, scale=0.31, seed=14)
    decode([70, 200], 4, 2, 96, 16, E4M3, q_extra=8, scale=0.31, seed=15)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_every_code_is_widened_exactly(dtype):
    """One token: the output is its V row, so each code's value times a scale of 1, rounded to bf16 (exact)."""
    dim, page = 256, 16
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    if dtype == E4M3:
        codes = torch.where((codes & 127) == 127, torch.zeros_like(codes), codes)      # NaN is not stored
    pool = torch.zeros(1, 2, 1, page, dim, device="cuda", dtype=torch.uint8)
    pool[0, 1, 0, 0] = codes
    pool[0, 0, 0, 0] = codes
    scales = torch.ones(1, 2, 1, page, device="cuda")
    q = torch.zeros(1, 1, dim, device="cuda").bfloat16()
    at = 3
    q[0, 0, at] = 1.0
    plan = ct.GqaPlan(ct.GqaLayout(1, dim, page, dtype, 1, 1), 1, 1, scale=1.0)
    out = torch.empty(1, 1, dim, device="cuda").bfloat16()
    lse = torch.empty(1, 1, device="cuda")
    for at in (3, 100, 250):                          # and the score is the K value it points at
        q.zero_()
        q[0, 0, at] = 1.0
        plan.decode(q, pool, scales, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                    torch.ones(1, dtype=torch.int32, device="cuda"), out, lse, stream=stream())
        torch.cuda.synchronize()
        want = (codes.view(torch.int8) if dtype == INT8 else codes.view(torch.float8_e4m3fn)).double()
        assert torch.equal(out[0, 0].double(), want)
        assert abs(float(lse[0, 0]) - float(want[at])) <= 2.0 ** -22 * abs(float(want[at])) + 1e-30


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_decode_values_of_very_different_size(dtype):
    """Queries, keys and values spread over many binary orders (the e4m3 path works with shifted exponents)."""
    g = gen(21)
    dim, page, n = 64, 16, 200
    table, n_pages = G.make_table([n], page, g)
    pool, scales = G.make_pool(n_pages, 1, page, dim, dtype, g)
    spread = torch.exp2(torch.randint(-12, 13, (n_pages, 2, 1, page), generator=g, device="cuda").float())
    if dtype == BF16:
        pool = (pool.float() * spread[..., None]).bfloat16()
    else:
        scales = scales * spread
    q = (torch.randn(1, 4, dim, generator=g, device="cuda")
         * torch.exp2(torch.randint(-18, 2, (1, 4, dim), generator=g, device="cuda").float())
         * torch.tensor([1.0, 2.0 ** -30, 2.0 ** -8, 2.0 ** -4], device="cuda")[None, :, None]).bfloat16()
    plan = ct.GqaPlan(ct.GqaLayout(1, dim, page, dtype, n_pages, table.shape[1]), 1, 4, scale=2.0 ** -6)
    out = torch.empty(1, 4, dim, device="cuda").bfloat16()
    lse = torch.empty(1, 4, device="cuda")
    plan.decode(q, pool, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), out, lse, stream=stream())
    torch.cuda.synchronize()
    ref = G.attend(q, pool, scales, table, [n], dtype, 4, MOD, scale=2.0 ** -6)
    G.check_attention(out, lse, ref, dim, n, dtype)


@pytest.mark.parametrize("dtype", [BF16, INT8])
def test_attended_nan_reaches_the_output(dtype):
    g = gen(22)
    table, n_pages = G.make_table([40, 40], 16, g)
    pool, scales = G.make_pool(n_pages, 1, 16, 64, dtype, g)
    (pool if dtype == BF16 else scales)[int(table[0, 1]), 0, 0, 3] = float("nan")
    q = torch.randn(2, 2, 64, generator=g, device="cuda").bfloat16()
    plan = ct.GqaPlan(ct.GqaLayout(1, 64, 16, dtype, n_pages, 3), 2, 2)
    out = torch.empty(2, 2, 64, device="cuda").bfloat16()
    plan.decode(q, pool, scales, table, torch.tensor([40, 40], dtype=torch.int32, device="cuda"), out, stream=stream())
    torch.cuda.synchronize()
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_pool_beyond_32_bit_offsets():
    g = gen(23)
    heads, dim, page, n_pages = 8, 128, 64, 18000                     # 2.36e9 values
    pool = torch.zeros(n_pages, 2, heads, page, dim, device="cuda", dtype=torch.bfloat16)
    pages = torch.tensor([[n_pages - 1, n_pages - 2, 17000]], dtype=torch.int32, device="cuda")
    pool[pages[0].long()] = torch.randn(3, 2, heads, page, dim, generator=g, device="cuda").bfloat16()
    q = torch.randn(1, 16, dim, generator=g, device="cuda").bfloat16()
    layout = ct.GqaLayout(heads, dim, page, BF16, n_pages, 3)
    plan = ct.GqaPlan(layout, 1, 16)
    out = torch.empty(1, 16, dim, device="cuda").bfloat16()
    lse = torch.empty(1, 16, device="cuda")
    plan.decode(q, pool, None, pages, torch.tensor([180], dtype=torch.int32, device="cuda"), out, lse, stream=stream())
    torch.cuda.synchronize()
    G.check_attention(out, lse, G.attend(q, pool, None, pages, [180], BF16, 16, MOD), dim, 180, BF16)
    rows = torch.randn(1, 2, heads * dim, generator=g, device="cuda").bfloat16()
    slot = torch.tensor([n_pages * page - 1], dtype=torch.int32, device="cuda")
    ct.gqa_write_slots(layout, pool, None, rows[:, 0], rows[:, 1], slot, 1, stream=stream())
    back = torch.empty(2, heads * dim, device="cuda").bfloat16()
    ct.gqa_read_slots(layout, pool, None, slot, 1, back[0], back[1], stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(pool[-1, :, :, -1], rows.view(2, heads, dim)) and torch.equal(back, rows[0])


# ---- write, read back, bounds ----------------------------------------------------------------------------------------

def written(heads, dim, page, dtype, n, src, fused, seed, special=True):
    g = gen(seed)
    n_pages = n // page + 3
    pool = torch.randint(0, 100, (n_pages, 2, heads, page, dim), generator=g, device="cuda")
    pool = pool.to({BF16: torch.bfloat16, INT8: torch.int8, E4M3: torch.uint8}[dtype])
    scales = None if dtype == BF16 else torch.full((n_pages, 2, heads, page), 3.0, device="cuda")
    width = heads * dim
    rows = torch.randn(n, 2 * width + (4 * width if fused else 0), generator=g, device="cuda")
    if special:
        rows[0] = 0.0
        if n > 5:
            rows[1, 5] = float("nan")
            rows[2, width + 1] = float("inf")
            rows[3] *= 1e30
            rows[4] *= 1e-39
            rows[5] = rows[5].abs() * 1e-42
    rows = rows if src == ct.CT_KV_F32 else rows.bfloat16()
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:n].to(torch.int32)
    if special and n > 9:
        slots[7], slots[8] = -1, n_pages * page
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, 4)
    return layout, pool, scales, rows, rows[:, :width], rows[:, width:2 * width], slots


@pytest.mark.parametrize("src", [BF16, ct.CT_KV_F32])
@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("heads,dim,page,n,fused", [(1, 32, 16, 1, False), (3, 96, 16, 77, True), (8, 128, 64, 300, True),
                                                    (2, 64, 48, 1000, False), (5, 192, 32, 40, False), (4, 256, 128, 65, True)])
def test_write_and_read_back_are_exact(heads, dim, page, n, fused, dtype, src):
    layout, pool, scales, rows, k, v, slots = written(heads, dim, page, dtype, n, src, fused, seed=n)
    want_pool, want_scales = pool.clone(), None if scales is None else scales.clone()
    sl = slots.cpu().numpy()
    ok = np.flatnonzero((sl >= 0) & (sl < pool.shape[0] * page))
    x = torch.stack((k, v), 1).float().cpu().numpy().reshape(n, 2, heads, dim)[ok]
    pg, st = torch.from_numpy(sl[ok] // page).long().cuda(), torch.from_numpy(sl[ok] % page).long().cuda()
    if dtype == BF16:
        want_pool.permute(0, 3, 1, 2, 4)[pg, st] = torch.from_numpy(x).cuda().bfloat16()
    else:
        codes, sc = G.encode(x, dtype)
        want_pool.permute(0, 3, 1, 2, 4)[pg, st] = torch.from_numpy(codes).cuda()
        want_scales.permute(0, 3, 1, 2)[pg, st] = torch.from_numpy(sc).cuda()
    ct.gqa_write_slots(layout, pool, scales, k, v, slots, n, src_dtype=src, k_stride=rows.shape[1], v_stride=rows.shape[1],
                       stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(pool.view(torch.uint8), want_pool.view(torch.uint8)) or (      # NaN rows of bf16: any NaN
        dtype == BF16 and torch.equal(torch.isnan(pool), torch.isnan(want_pool))
        and torch.equal(pool.nan_to_num(), want_pool.nan_to_num()))
    if scales is not None:
        assert torch.equal(torch.isnan(scales), torch.isnan(want_scales))
        assert torch.equal(scales.nan_to_num(), want_scales.nan_to_num())
    for out_dtype, t in ((BF16, torch.bfloat16), (ct.CT_KV_F32, torch.float32)):
        kb = torch.full((n, heads * dim + 8), 5.0, device="cuda").to(t)
        vb = torch.full((n, heads * dim), 5.0, device="cuda").to(t)
        ct.gqa_read_slots(layout, pool, scales, slots, n, kb, vb, out_dtype=out_dtype, k_stride=heads * dim + 8, stream=stream())
        torch.cuda.synchronize()
        assert (kb[:, heads * dim:] == 5.0).all()
        skipped = np.setdiff1d(np.arange(n), ok)
        assert (kb[skipped] == 5.0).all() and (vb[skipped] == 5.0).all()
        stored = pool.permute(0, 3, 1, 2, 4)[pg, st].contiguous()
        if dtype == BF16:
            want = stored.float()
        else:
            c = stored.float() if dtype == INT8 else stored.view(torch.float8_e4m3fn).float()
            want = c * scales.permute(0, 3, 1, 2)[pg, st][..., None]                  # one fp32 rounding
        want = want.to(t).reshape(len(ok), 2, heads * dim)
        got = torch.stack((kb[ok][:, :heads * dim], vb[ok]), 1)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("heads,dim,page", [(1, 32, 16), (3, 96, 48), (8, 128, 64), (2, 256, 128), (4, 192, 32), (2, 64, 64)])
def test_page_bounds_are_exact(heads, dim, page, dtype):
    g = gen(31)
    n_pages = 9
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    pool[2, 0] = 0
    (pool if dtype == BF16 else scales)[3, 0, 0, 1] = float("nan")
    (pool if dtype == BF16 else scales)[4, 0, :, page // 2:] = float("nan")           # behind the count
    if dtype == BF16:
        pool[5, 0, 0, 0, 3] = float("inf")
    pages = torch.tensor([0, 1, 2, 3, 4, 5, 6, -1, 9, 8], dtype=torch.int32, device="cuda")
    counts = torch.tensor([page, 1, page, page, page // 2, 5, 0, 4, 4, page + 7], dtype=torch.int32, device="cuda")
    bounds = torch.full((n_pages, heads, 2, dim), 9, dtype=torch.int8, device="cuda")
    bs = torch.full((n_pages, heads), 9.0, device="cuda")
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, 4)
    ct.gqa_page_bounds(layout, pool, scales, pages, counts, 10, bounds, bs, stream=stream())
    torch.cuda.synchronize()
    assert (bounds[7] == 9).all() and (bs[7] == 9).all()                              # not listed
    if dtype == BF16:
        k = pool[:, 0].float().cpu().numpy()
    else:
        c = pool[:, 0].float() if dtype == INT8 else pool[:, 0].contiguous().view(torch.float8_e4m3fn).float()
        k = (c * scales[:, 0][..., None]).cpu().numpy()
    for p, n in ((0, page), (1, 1), (2, page), (3, page), (4, page // 2), (5, 5), (6, 0), (8, page)):
        for h in range(heads):
            codes, s = G.bounds_of(k[p, h, :n])
            assert np.array_equal(bounds[p, h].cpu().numpy(), codes), (p, h)
            assert np.array_equal(np.float32(bs[p, h].item()), s, equal_nan=True), (p, h)


# ---- selection ----------------------------------------------------------------------------------------------------------

def selection(lens, heads, group, dim, page, n_select, first=1, last=1, order=MOD, window=0, seed=41, holes=(), edit=None,
              q_extra=0):
    g = gen(seed)
    table, n_pages = G.make_table(lens, page, g, window, holes=holes)
    bounds = torch.randint(-127, 128, (n_pages, heads, 2, dim), generator=g, device="cuda", dtype=torch.int8)
    bounds = bounds.sort(2, descending=True).values.contiguous()
    bs = torch.rand(n_pages, heads, generator=g, device="cuda") + 0.1
    hq = heads * group
    q = torch.randn(len(lens), hq * dim + q_extra, generator=g, device="cuda").bfloat16()
    if edit:
        edit(q, bounds, bs, table)
    plan = ct.GqaPlan(ct.GqaLayout(heads, dim, page, BF16, n_pages, table.shape[1]), len(lens), hq, window_tokens=window,
                      head_order=order)
    got = torch.full((len(lens), heads, n_select), 77, dtype=torch.int32, device="cuda")
    plan.select(q, bounds, bs, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), got, n_select, first, last,
                q_stride=q.shape[1], stream=stream())
    torch.cuda.synchronize()
    qv = q[:, :hq * dim].float().cpu().numpy().reshape(len(lens), hq, dim)
    want = G.select(qv, bounds.cpu().numpy(), bs.cpu().numpy(), table.cpu().numpy(), lens, n_pages, page, hq, order, n_select,
                    first, last, window)
    assert np.array_equal(got.cpu().numpy(), want)
    return got


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_selection_is_exact(dim):
    selection([0, 1, 64, 65, 1000, 5000, 4097], 2, 4, dim, 64, 8, seed=dim)


@pytest.mark.parametrize("group,order", [(1, MOD), (7, BLK), (16, MOD), (17, BLK), (40, MOD)])
def test_selection_groups(group, order):
    selection([900, 3000], 3, group, 64, 16, 11, order=order, seed=group, q_extra=64)


@pytest.mark.parametrize("n_select,first,last", [(1, 0, 0), (1, 1, 0), (2, 1, 1), (5, 2, 3), (64, 0, 4), (500, 3, 0), (255, 1, 1)])
def test_selection_counts(n_select, first, last):
    selection([16 * 300, 16 * 255, 37, 16 * 256 + 1], 2, 2, 64, 16, n_select, first, last, seed=n_select)


def test_selection_window_and_unmapped_pages():
    selection([2000, 700, 5000], 2, 2, 64, 32, 6, window=1000, seed=3)
    holes = {(0, i) for i in range(0, 60, 2)} | {(1, i) for i in range(22)}
    got = selection([2000, 700, 5000], 2, 2, 64, 32, 40, holes=holes, seed=4)
    assert (got[1] == -1).all()                       # a sequence without mapped pages


def test_selection_ties_go_to_the_lowest_page():
    def same(q, bounds, bs, table):
        bounds[:] = bounds[:1]
        bs[:] = 0.5
    got = selection([64 * 50], 2, 3, 128, 64, 9, edit=same)
    assert got[0, 0].tolist() == list(range(8)) + [49]

    def zeros(q, bounds, bs, table):
        q.zero_()
        bs[table[0, 5].long()] = 0.0
    selection([64 * 50], 2, 3, 128, 64, 9, edit=zeros)


def test_selection_of_scores_that_are_not_numbers():
    def nan_page(q, bounds, bs, table):
        bs[table[0, 17].long(), 0] = float("nan")
    got = selection([64 * 50], 2, 3, 128, 64, 4, edit=nan_page)
    assert 17 in got[0, 0].tolist()

    def nan_query(q, bounds, bs, table):
        q[0, 3] = float("nan")
        q[1, 128 * 4] = float("inf")
    selection([64 * 50, 64 * 40], 2, 3, 128, 64, 4, edit=nan_query)


def test_selection_of_a_very_long_sequence():
    selection([16 * 20011, 16 * 49152], 1, 2, 32, 16, 1000, seed=8)


# ---- decode over selected pages ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("heads,group,dim,page,pick,window", [(2, 4, 128, 64, 5, 0), (1, 16, 64, 16, 7, 300), (3, 1, 96, 48, 1, 0),
                                                              (1, 20, 256, 128, 3, 0), (2, 2, 32, 32, 40, 0)])
def test_decode_selected(heads, group, dim, page, pick, window, dtype):
    g = gen(51 + dim)
    lens = [900, 0, 1, 333, 1500]
    table, n_pages = G.make_table(lens, page, g, window)
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    tb = table.cpu().numpy()
    for s, n in enumerate(lens):
        if n % page:
            (pool if dtype == BF16 else scales)[int(tb[s, n // page]), :, :, n % page:] = float("nan")
    rng = np.random.default_rng(3)
    pages = np.full((len(lens), heads, pick), -1, np.int32)
    for s, n in enumerate(lens):
        have = np.flatnonzero(tb[s] >= 0)
        for h in range(heads):
            sel = np.sort(rng.permutation(have)[:pick])
            pages[s, h, :len(sel)] = sel
    hq = heads * group
    q = torch.randn(len(lens), hq, dim, generator=g, device="cuda").bfloat16()
    plan = ct.GqaPlan(ct.GqaLayout(heads, dim, page, dtype, n_pages, table.shape[1]), len(lens), hq, window_tokens=window)
    out = torch.empty(len(lens), hq, dim, device="cuda").bfloat16()
    lse = torch.empty(len(lens), hq, device="cuda")
    plan.decode_selected(q, pool, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(pages).cuda(), pick, out, lse, stream=stream())
    torch.cuda.synchronize()
    ref = G.attend(q, pool, scales, table, lens, dtype, hq, MOD, window, pages=pages)
    G.check_attention(out, lse, ref, dim, max(lens), dtype)


def test_decode_selected_ignores_pages_outside_the_sequence():
    g = gen(61)
    lens, page = [300, 100], 64
    table, n_pages = G.make_table(lens, page, g, holes={(0, 2)})
    pool, _ = G.make_pool(n_pages, 1, page, 64, BF16, g)
    pages = np.array([[[0, 2, 4, 5000]], [[1, 3, -7, -1]]], np.int32)                 # 2: unmapped; 3 and 5000: not its own
    q = torch.randn(2, 3, 64, generator=g, device="cuda").bfloat16()
    plan = ct.GqaPlan(ct.GqaLayout(1, 64, page, BF16, n_pages, table.shape[1]), 2, 3)
    out = torch.empty(2, 3, 64, device="cuda").bfloat16()
    lse = torch.empty(2, 3, device="cuda")
    plan.decode_selected(q, pool, None, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(pages).cuda(), 4, out, lse, stream=stream())
    torch.cuda.synchronize()
    G.check_attention(out, lse, G.attend(q, pool, None, table, lens, BF16, 3, MOD, pages=pages), 64, 300, BF16)


# ---- the handle, and the operators together -----------------------------------------------------------------------------------

def rows(n, heads, dim, g):
    return torch.randn(2, n, heads * dim, generator=g, device="cuda").bfloat16()


def stored_as(x, dtype, heads, dim):
    """What bf16 rows [n][heads * dim] read back as in fp32."""
    if dtype == BF16:
        return x.float()
    codes, sc = G.encode(x.float().cpu().numpy().reshape(-1, heads, dim), dtype)
    c = torch.from_numpy(codes)
    c = c.float() if dtype == INT8 else c.view(torch.float8_e4m3fn).float()
    return (c * torch.from_numpy(sc)[..., None]).reshape(x.shape[0], -1).cuda()


def recomputed_bounds(kv, heads, dim, page, dtype):
    """Codes and scales that a fresh pass over the handle's pages gives, for its mapped pages."""
    lay = kv.layout
    lens, tb = kv.seq_lens(), kv.block_table()
    pages = {}
    for s in range(len(lens)):
        for lp in range(tb.shape[1]):
            if tb[s, lp] >= 0:
                pages[int(tb[s, lp])] = min(page, int(lens[s]) - lp * page)
    ids = torch.tensor(list(pages), dtype=torch.int32, device="cuda")
    cnt = torch.tensor(list(pages.values()), dtype=torch.int32, device="cuda")
    b = torch.zeros(lay.n_pages, heads, 2, dim, dtype=torch.int8, device="cuda")
    s = torch.zeros(lay.n_pages, heads, device="cuda")
    ct.gqa_page_bounds(lay, kv.pool, kv.scales, ids, cnt, len(pages), b, s, stream=stream())
    torch.cuda.synchronize()
    return ids.long(), b, s


def dev_copy(addr, shape, t):
    out = torch.empty(shape, dtype=t, device="cuda")
    ct.check(ct.lib().ct_hal_cuda_memcpy(out.data_ptr(), addr, out.numel() * out.element_size(), 2, stream()))
    torch.cuda.synchronize()
    return out


def check_bounds(kv, heads, dim, page, dtype):
    ids, b, s = recomputed_bounds(kv, heads, dim, page, dtype)
    assert torch.equal(dev_copy(kv.bounds, b.shape, torch.int8)[ids], b[ids])
    assert torch.equal(dev_copy(kv.bound_scales, s.shape, torch.float32)[ids], s[ids])


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_handle_append_fork_compact_checkpoint(dtype, tmp_path):
    heads, dim, page = 3, 64, 16
    g = gen(71)
    kv = ct.GqaKV(4, 40, 60, heads, dim, page, dtype=dtype, keep_bounds=True, stream=stream())
    rng = np.random.default_rng(5)
    kv.set_free_order(rng.permutation(60))
    hist = {s: [] for s in range(4)}
    for counts in ([5, 40, 0], [1, 1, 1], [33, 0, 100], [1, 1, 1]):
        x = rows(sum(counts), heads, dim, g)
        kv.append_kv([0, 1, 2], counts, x[0], x[1])
        at = 0
        for s, c in zip((0, 1, 2), counts):
            hist[s].append(x[:, at:at + c])
            at += c
    check_bounds(kv, heads, dim, page, dtype)
    kv.fork(1, 3, 37)                                 # two shared pages and a copied partial one
    hist[3] = [torch.cat(hist[1], 1)[:, :37]]
    check_bounds(kv, heads, dim, page, dtype)
    x = rows(3, heads, dim, g)
    kv.append_kv([3], [3], x[0], x[1])
    hist[3].append(x)
    entries = torch.cat((x[0], x[1]), 1).contiguous()                                # the same call with whole entries
    kv.append([0], [3], entries)
    hist[0].append(x)
    check_bounds(kv, heads, dim, page, dtype)

    def same(h):
        lens = h.seq_lens()
        n = int(lens.sum())
        k, v = (torch.empty(n, heads * dim, device="cuda") for _ in range(2))
        h.gather_kv(range(4), [0] * 4, lens, k, v, ct.CT_KV_F32)
        whole = torch.empty(n, 2 * heads * dim, device="cuda")
        h.gather_batch(range(4), [0] * 4, lens, whole, ct.CT_KV_F32)
        one = torch.empty(20, 2 * heads * dim, device="cuda").bfloat16()
        h.gather(1, 7, 20, one)
        torch.cuda.synchronize()
        want = torch.cat([torch.cat(hist[s], 1) for s in range(4)], 1)
        wk, wv = stored_as(want[0], dtype, heads, dim), stored_as(want[1], dtype, heads, dim)
        assert torch.equal(k, wk) and torch.equal(v, wv)
        assert torch.equal(whole, torch.cat((wk, wv), 1))
        a = int(lens[0]) + 7
        assert torch.equal(one, torch.cat((wk, wv), 1)[a:a + 20].bfloat16())

    same(kv)
    kv.compact()
    same(kv)
    check_bounds(kv, heads, dim, page, dtype)
    kv.compact()
    kv.save(tmp_path / "c.bin")
    back = ct.GqaKV.load(tmp_path / "c.bin", stream=stream())
    assert back.layout.n_kv_heads == heads and back.layout.head_dim == dim and back.layout.kv_dtype == dtype
    same(back)
    check_bounds(back, heads, dim, page, dtype)
    x = rows(1, heads, dim, g)
    for h in (kv, back):
        h.append_kv([2], [1], x[0], x[1])
    hist[2].append(x)
    same(kv)
    same(back)


def test_handle_window_and_eviction_keep_bounds():
    heads, dim, page = 2, 128, 16
    g = gen(72)
    kv = ct.GqaKV(3, 200, 14, heads, dim, page, window_tokens=100, dtype=INT8, keep_bounds=True, stream=stream())
    for step in range(40):
        counts = [7, 1, step % 3]
        x = rows(sum(counts), heads, dim, g)
        kv.append_kv([0, 1, 2], counts, x[0], x[1])
    assert kv.stats().n_evict_window > 0
    check_bounds(kv, heads, dim, page, INT8)


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_serving_steps_append_select_decode(dtype):
    """Growing sequences: K and V appended through the handle, pages chosen, attention over them, and over everything."""
    heads, group, dim, page, pick = 2, 4, 128, 16, 6
    hq = heads * group
    g = gen(73)
    kv = ct.GqaKV(3, 64, 150, heads, dim, page, dtype=dtype, keep_bounds=True, stream=stream())
    x = rows(700, heads, dim, g)
    kv.append_kv([0, 1, 2], [400, 5, 295], x[0], x[1])
    plan = ct.GqaPlan(kv.layout, 3, hq)
    fused = torch.empty(3, (hq + 2 * heads) * dim, device="cuda").bfloat16()
    picked = torch.empty(3, heads, pick, dtype=torch.int32, device="cuda")
    out, out_sel = (torch.empty(3, hq, dim, device="cuda").bfloat16() for _ in range(2))
    lse, lse_sel = (torch.empty(3, hq, device="cuda") for _ in range(2))
    NP = kv.layout.n_pages

    def attend():
        st = torch.cuda.current_stream().cuda_stream
        plan.select(fused, kv.bounds, kv.bound_scales, kv.block_table_dev, kv.seq_lens_dev, picked, pick,
                    q_stride=fused.shape[1], stream=st)
        plan.decode_selected(fused, kv.pool, kv.scales, kv.block_table_dev, kv.seq_lens_dev, picked, pick, out_sel, lse_sel,
                             q_stride=fused.shape[1], stream=st)
        plan.decode(fused, kv.pool, kv.scales, kv.block_table_dev, kv.seq_lens_dev, out, lse, q_stride=fused.shape[1],
                    stream=st)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend()
    for step in range(20):
        fused.copy_(torch.randn(fused.shape, generator=g, device="cuda"))
        kv.append_kv([0, 1, 2], [1, 1, 1], fused[:, hq * dim:], fused[:, (hq + heads) * dim:], k_stride=fused.shape[1],
                     v_stride=fused.shape[1])
        graph.replay() if step % 2 else attend()
        torch.cuda.synchronize()
        if step not in (0, 1, 10, 19):
            continue
        lens, tb = kv.seq_lens().tolist(), torch.from_numpy(kv.block_table()).cuda()
        shape = (NP, 2, heads, page, dim)
        pool = dev_copy(kv.pool, shape, {BF16: torch.bfloat16, INT8: torch.int8, E4M3: torch.uint8}[dtype])
        scales = None if dtype == BF16 else dev_copy(kv.scales, shape[:4], torch.float32)
        q = fused[:, :hq * dim].reshape(3, hq, dim)
        bounds = dev_copy(kv.bounds, (NP, heads, 2, dim), torch.int8).cpu().numpy()
        bs = dev_copy(kv.bound_scales, (NP, heads), torch.float32).cpu().numpy()
        want = G.select(q.float().cpu().numpy(), bounds, bs, tb.cpu().numpy(), lens, NP, page, hq, MOD, pick, 1, 1)
        assert np.array_equal(picked.cpu().numpy(), want)
        G.check_attention(out_sel, lse_sel, G.attend(q, pool, scales, tb, lens, dtype, hq, MOD, pages=want), dim, max(lens),
                          dtype)
        G.check_attention(out, lse, G.attend(q, pool, scales, tb, lens, dtype, hq, MOD), dim, max(lens), dtype)


def test_two_plans_on_two_streams():
    g = gen(74)
    lens = [5000, 70]
    table, n_pages = G.make_table(lens, 64, g)
    pool, _ = G.make_pool(n_pages, 2, 64, 128, BF16, g)
    q = torch.randn(2, 2, 8, 128, generator=g, device="cuda").bfloat16()
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    layout = ct.GqaLayout(2, 128, 64, BF16, n_pages, table.shape[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    plans = [ct.GqaPlan(layout, 2, 8) for _ in range(2)]
    outs = torch.zeros(2, 2, 8, 128, device="cuda").bfloat16()
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            plans[i].decode(q[i], pool, None, table, ld, outs[i], stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        G.check_attention(outs[i], None, G.attend(q[i], pool, None, table, lens, BF16, 8, MOD), 128, 5000, BF16)


def test_results_do_not_change_from_run_to_run():
    """Joins go by index, never by arrival: the same bits on every run."""
    g = gen(75)
    lens = [9000, 1, 777, 3001]
    table, n_pages = G.make_table(lens, 64, g)
    pool, scales = G.make_pool(n_pages, 2, 64, 128, E4M3, g)
    q = torch.randn(4, 8, 128, generator=g, device="cuda").bfloat16()
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    plan = ct.GqaPlan(ct.GqaLayout(2, 128, 64, E4M3, n_pages, table.shape[1]), 4, 8)
    first = None
    for _ in range(30):
        out = torch.empty(4, 8, 128, device="cuda").bfloat16()
        lse = torch.empty(4, 8, device="cuda")
        plan.decode(q, pool, scales, table, ld, out, lse, stream=stream())
        torch.cuda.synchronize()
        if first is None:
            first = (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_nothing_to_do():
    layout = ct.GqaLayout(1, 64, 16, BF16, 4, 2)
    plan = ct.GqaPlan(layout, 0, 1)
    t = torch.zeros(64, device="cuda")
    plan.decode(t, t, None, t, t, t, stream=stream())
    plan.select(t, t, t, t, t, t, 2, stream=stream())
    ct.gqa_write_slots(layout, t, None, t, t, t, 0, stream=stream())
    ct.gqa_read_slots(layout, t, None, t, 0, t, t, stream=stream())
    ct.gqa_page_bounds(layout, t, None, t, t, 0, t, t, stream=stream())
    torch.cuda.synchronize()


def test_plan_refusals_on_the_device():
    layout = ct.GqaLayout(2, 64, 16, INT8, 4, 2)
    plan = ct.GqaPlan(layout, 1, 4)
    t = torch.zeros(4096, device="cuda")
    L, a = ct.lib(), t.data_ptr()
    dec = lambda p=plan.h, q=a, qs=0, pool=a, sc=a, bt=a, ln=a, out=a: L.ct_attn_gqa_decode_paged(p, q, qs, pool, sc, bt, ln, out, None, None)  # noqa: E731
    for bad in (dict(p=None), dict(q=None), dict(q=a + 8), dict(qs=128), dict(qs=257), dict(pool=None), dict(pool=a + 4),
                dict(sc=None), dict(sc=a + 4), dict(bt=None), dict(ln=None), dict(out=None), dict(out=a + 2)):
        assert dec(**bad) == ct.CT_ERR_ARG, bad
    sel = lambda n=2, f=1, l=1, b=a, o=a: L.ct_attn_gqa_select_pages(plan.h, a, 0, b, a, a, a, n, f, l, o, None)  # noqa: E731
    for bad in (dict(n=0, f=0, l=0), dict(n=1), dict(f=0xFFFFFFFF), dict(b=None), dict(b=a + 8), dict(o=None)):
        assert sel(**bad) == ct.CT_ERR_ARG, bad
    assert L.ct_attn_gqa_decode_selected(plan.h, a, 0, a, a, a, a, None, 2, a, None, None) == ct.CT_ERR_ARG
    assert L.ct_attn_gqa_decode_selected(plan.h, a, 0, a, a, a, a, a, 0, a, None, None) == ct.CT_ERR_ARG
    far = ct.GqaPlan(ct.GqaLayout(1, 64, 16, BF16, 4, 49153), 1, 1)
    assert L.ct_attn_gqa_select_pages(far.h, a, 0, a, a, a, a, 2, 1, 1, a, None) == ct.CT_ERR_UNSUPPORTED


def test_page_bounds_see_not_a_number_codes():
    """An e4m3 pool that another program filled may hold the format's NaN codes."""
    g = gen(81)
    heads, dim, page = 2, 96, 32
    pool, scales = G.make_pool(4, heads, page, dim, E4M3, g)
    raw = pool.view(torch.uint8)
    raw[1, 0, 0, 3, 95] = 0x7F                                # page 1, head 0
    raw[2, 0, 1, 31, 0] = 0xFF                                # page 2, head 1
    raw[3, 0, 0, 20, 1] = 0x7F                                # behind the count
    raw[3, 1, 1, 0, 1] = 0x7F                                 # a value, not a key
    bounds = torch.zeros(4, heads, 2, dim, dtype=torch.int8, device="cuda")
    bs = torch.zeros(4, heads, device="cuda")
    ct.gqa_page_bounds(ct.GqaLayout(heads, dim, page, E4M3, 4, 4), pool, scales,
                       torch.arange(4, dtype=torch.int32, device="cuda"),
                       torch.tensor([32, 32, 32, 20], dtype=torch.int32, device="cuda"), 4, bounds, bs, stream=stream())
    torch.cuda.synchronize()
    assert torch.isnan(bs).tolist() == [[False, False], [True, False], [False, True], [False, False]]
    assert (bounds[1, 0] == 0).all() and (bounds[2, 1] == 0).all()


@pytest.mark.parametrize("dtype,dim,group", [(BF16, 128, 4), (INT8, 128, 16), (E4M3, 64, 1)])
def test_decode_one_long_sequence_among_many_short(dtype, dim, group):
    """The long one's items span so many CTAs that their parts are joined in two rounds, beside whole items."""
    lens = [(i * 7) % 20 for i in range(150)] + [60000] + [(i * 5) % 33 for i in range(150)]
    decode(lens, 2, group, dim, 64, dtype, seed=82)


def test_decode_thousands_of_sequences():
    lens = [(i * 29) % 41 for i in range(5000)]
    decode(lens, 2, 2, 64, 16, INT8, seed=83)
    decode(lens[:3000], 1, 8, 128, 32, BF16, seed=84)


def test_selection_shared_by_a_cluster():
    """Few rows of many pages: several CTAs score one row, for groups of one and of several head tiles."""
    selection([16 * 4000 + 3, 16 * 700], 1, 33, 128, 16, 40, seed=85)
    selection([16 * 3000], 2, 5, 64, 16, 9, first=0, last=3, window=16 * 2000 + 5, seed=86)


@pytest.mark.parametrize("dtype", [BF16, INT8])
def test_captured_calls_share_a_plan_and_follow_the_lengths(dtype):
    """Two graphs over one plan, replayed in turn on one stream after the lengths changed, rows of the padded batch empty;
    and one graph of another plan beside them on a second stream."""
    g = gen(87)
    heads, group, dim, page, S = 2, 4, 128, 64, 5
    hq = heads * group
    longest = [9000, 600, 64, 3000, 1]
    table, n_pages = G.make_table(longest, page, g)
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, table.shape[1])
    plan, other = ct.GqaPlan(layout, S, hq), ct.GqaPlan(layout, S, hq)
    q = torch.randn(3, S, hq, dim, generator=g, device="cuda").bfloat16()
    lens = torch.tensor(longest, dtype=torch.int32, device="cuda")
    out = torch.zeros(3, S, hq, dim, device="cuda").bfloat16()
    lse = torch.zeros(3, S, hq, device="cuda")
    side = torch.cuda.Stream()
    graphs = []
    for i, p in enumerate((plan, plan, other)):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(3):
                p.decode(q[i], pool, scales, table, lens, out[i], lse[i], stream=torch.cuda.current_stream().cuda_stream)
    for now in ([9000, 600, 64, 3000, 1], [0, 0, 0, 17, 0], [8999, 0, 0, 0, 0], [0] * 5, [5, 600, 1, 2999, 0]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(4):
            graphs[0].replay()
            graphs[1].replay()
            with torch.cuda.stream(side):
                graphs[2].replay()
        torch.cuda.synchronize()
        for i in range(3):
            G.check_attention(out[i], lse[i], G.attend(q[i], pool, scales, table, now, dtype, hq, MOD), dim, max(max(now), 1),
                              dtype)


def test_captured_write_bounds_and_read_follow_the_slots():
    """One token a sequence as in a decode step, captured once; the padded rows' slots are outside the pool."""
    g = gen(88)
    heads, dim, page, n_pages, S = 3, 64, 32, 6, 4
    layout = ct.GqaLayout(heads, dim, page, INT8, n_pages, 4)
    pool = torch.zeros(n_pages, 2, heads, page, dim, dtype=torch.int8, device="cuda")
    scales = torch.zeros(n_pages, 2, heads, page, device="cuda")
    bounds = torch.zeros(n_pages, heads, 2, dim, dtype=torch.int8, device="cuda")
    bs = torch.zeros(n_pages, heads, device="cuda")
    x = torch.zeros(S, 2 * heads * dim, device="cuda").bfloat16()
    back = torch.full((2, S, heads * dim), 5.0, device="cuda").bfloat16()
    slots = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    pages, counts = (torch.full((S,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        ct.gqa_write_slots(layout, pool, scales, x, x[:, heads * dim:], slots, S, k_stride=2 * heads * dim,
                           v_stride=2 * heads * dim, stream=st)
        ct.gqa_page_bounds(layout, pool, scales, pages, counts, S, bounds, bs, stream=st)
        ct.gqa_read_slots(layout, pool, scales, slots, S, back[0], back[1], stream=st)
    kept = torch.zeros(2 * page, heads, dim)
    for step in range(2 * page):                              # sequence 0 fills page 4, then page 1
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        page_now, at = (4, step) if step < page else (1, step - page)
        slots.copy_(torch.tensor([page_now * page + at, -1, n_pages * page, -7], dtype=torch.int32))
        pages.copy_(torch.tensor([page_now, -1, n_pages, -2], dtype=torch.int32))
        counts.copy_(torch.tensor([at + 1, 3, 3, 3], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        codes, sc = G.encode(x[0].float().cpu().numpy().reshape(2 * heads, dim), INT8)
        want = np.asarray(codes, dtype=np.float32).reshape(2, heads, dim) * np.asarray(sc, dtype=np.float32).reshape(2, heads, 1)
        kept[step] = torch.from_numpy(want[0])
        assert torch.equal(back[:, 0].cpu(), torch.from_numpy(want).bfloat16().reshape(2, heads * dim))
        assert (back[:, 1:] == 5.0).all()
        for h in range(heads):
            run = kept[step - at:step + 1, h].numpy()
            want_codes, want_s = G.bounds_of(run)
            assert np.array_equal(bounds[page_now, h].cpu().numpy(), want_codes) and bs[page_now, h].item() == want_s


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (INT8, 128), (E4M3, 64)])
def test_decode_warps_that_pass_many_pages(dtype, dim):
    """Small pages and enough items that each warp's run of tokens goes over more than 64 of them, holes among them."""
    lens = [2900 + 13 * i for i in range(48)]
    holes = {(s, p) for s in range(0, 48, 5) for p in range(20, 80, 7)}
    decode(lens, 8, 1, dim, 16, dtype, holes=holes, seed=89)


@pytest.mark.parametrize("dtype,window", [(BF16, 0), (INT8, 3999)])
def test_decode_many_selected_pages(dtype, window):
    """Long lists of small pages: more entries than a warp loads at a time, sequences shorter than their list among them."""
    g = gen(90)
    heads, group, dim, page, pick, S = 4, 4, 128, 16, 220, 40
    lens = [5000 + 3 * i for i in range(S - 2)] + [700, 0]
    table, n_pages = G.make_table(lens, page, g, window)
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    q = torch.randn(S, heads * group, dim, generator=g, device="cuda").bfloat16()
    pages = np.full((S, heads, pick), -1, np.int32)
    rng = np.random.default_rng(5)
    for s, n in enumerate(lens):
        first, last = (max(0, n - window) // page if window else 0), -(-n // page)
        for h in range(heads):
            k = min(pick, last - first)
            pages[s, h, :k] = np.sort(rng.permutation(np.arange(first, last))[:k])
    plan = ct.GqaPlan(ct.GqaLayout(heads, dim, page, dtype, n_pages, table.shape[1]), S, heads * group, window_tokens=window)
    out = torch.empty(S, heads * group, dim, device="cuda").bfloat16()
    lse = torch.empty(S, heads * group, device="cuda")
    plan.decode_selected(q, pool, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(pages).cuda(), pick, out, lse, stream=stream())
    torch.cuda.synchronize()
    G.check_attention(out, lse, G.attend(q, pool, scales, table, lens, dtype, heads * group, MOD, window, pages=pages), dim,
                      max(lens), dtype)


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_calls_in_a_row_see_what_the_one_before_wrote(dtype):
    """Write, bounds, read back, selection, both decodes and a copy of the lengths, over the same buffers again and again
    without a wait: the bits of the same calls with a wait after each."""
    g = gen(91)
    heads, group, dim, page, S, pick, steps = 2, 4, 64, 16, 6, 3, 60
    hq, per, n_pages = heads * group, 12, 6 * 12
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, per)
    plan = ct.GqaPlan(layout, S, hq)
    n, width = S * page * 5, heads * dim
    x = torch.randn(steps, n, 2 * width, generator=g, device="cuda").bfloat16()
    q = torch.randn(steps, S, hq, dim, generator=g, device="cuda").bfloat16()
    tables = torch.stack([torch.randperm(n_pages, generator=g, device="cuda").view(S, per) for _ in range(steps)]).to(torch.int32)
    lens_bank = torch.randint(1, 5 * page + 1, (steps, S), generator=g, device="cuda").to(torch.int32)
    t = torch.arange(page * 5, device="cuda")
    slot_bank = (tables[:, :, t // page] * page + t % page).reshape(steps, n).to(torch.int32).contiguous()

    def run(wait):
        pool = torch.zeros(n_pages, 2, heads, page, dim, device="cuda",
                           dtype={BF16: torch.bfloat16, INT8: torch.int8, E4M3: torch.uint8}[dtype])
        scales = None if dtype == BF16 else torch.zeros(n_pages, 2, heads, page, device="cuda")
        bounds = torch.zeros(n_pages, heads, 2, dim, dtype=torch.int8, device="cuda")
        bs = torch.zeros(n_pages, heads, device="cuda")
        pages = torch.arange(n_pages, dtype=torch.int32, device="cuda")
        counts = torch.full((n_pages,), page, dtype=torch.int32, device="cuda")
        slots, table, lens, picked = slot_bank[0].clone(), tables[0].clone(), lens_bank[0].clone(), torch.zeros(
            S, heads, pick, dtype=torch.int32, device="cuda")
        back = torch.zeros(steps, 2, n, width, device="cuda")
        out = torch.zeros(steps, 2, S, hq, dim, device="cuda").bfloat16()
        chosen = torch.zeros(steps, S, heads, pick, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        for i in range(steps):
            def then():
                if wait:
                    torch.cuda.synchronize()
            slots.copy_(slot_bank[i]); then()  # noqa: E702
            ct.gqa_write_slots(layout, pool, scales, x[i], x[i, :, width:], slots, n, k_stride=2 * width, v_stride=2 * width,
                               stream=stream()); then()  # noqa: E702
            ct.gqa_page_bounds(layout, pool, scales, pages, counts, n_pages, bounds, bs, stream=stream()); then()  # noqa: E702
            ct.gqa_read_slots(layout, pool, scales, slots, n, back[i, 0], back[i, 1], out_dtype=ct.CT_KV_F32,
                              stream=stream()); then()  # noqa: E702
            table.copy_(tables[i]); lens.copy_(lens_bank[i]); then()  # noqa: E702
            plan.select(q[i], bounds, bs, table, lens, picked, pick, stream=stream()); then()  # noqa: E702
            plan.decode_selected(q[i], pool, scales, table, lens, picked, pick, out[i, 0], stream=stream()); then()  # noqa: E702
            plan.decode(q[i], pool, scales, table, lens, out[i, 1], stream=stream()); then()  # noqa: E702
            chosen[i].copy_(picked); then()  # noqa: E702
        torch.cuda.synchronize()
        return back, out, chosen

    want = run(True)
    for _ in range(3):
        for a, b in zip(run(False), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, INT8])
def test_fork_from_a_full_pool_keeps_the_source(dtype):
    """No page is free: another sequence gives one up, the fork reads what its source reads, and the source keeps its tokens."""
    heads, dim, page = 2, 64, 16
    g = gen(92)
    kv = ct.GqaKV(3, 8, 4, heads, dim, page, dtype=dtype, keep_bounds=True, stream=stream())
    x = rows(64, heads, dim, g)
    kv.append_kv([0, 2], [32, 32], x[0], x[1])
    kv.fork(0, 1, 5)
    got = torch.empty(2, 37, heads * dim, device="cuda")
    kv.gather_kv([0, 1], [0, 0], [32, 5], got[0], got[1], ct.CT_KV_F32)
    torch.cuda.synchronize()
    for i in range(2):
        want = stored_as(x[i], dtype, heads, dim)
        assert torch.equal(got[i], torch.cat((want[:32], want[:5])))
    assert ct.lib().ct_kv_paged_gather(kv.h, 2, 0, 1, got.data_ptr(), BF16) == ct.CT_ERR_UNMAPPED
    check_bounds(kv, heads, dim, page, dtype)


@pytest.mark.parametrize("dtype,page", [(BF16, 272), (INT8, 272), (INT8, 512), (E4M3, 512), (BF16, 512)])
def test_large_pages_append_compact_checkpoint_and_decode(dtype, page, tmp_path):
    heads, group, dim = 2, 4, 64
    hq = heads * group
    g = gen(page + dtype)
    kv = ct.GqaKV(3, 6, 12, heads, dim, page, dtype=dtype, keep_bounds=True, stream=stream())
    kv.set_free_order(np.random.default_rng(6).permutation(12))
    lens = [3 * page + 7, 1, 2 * page]
    x = rows(sum(lens), heads, dim, g)
    kv.append_kv([0, 1, 2], lens, x[0], x[1])
    wk, wv = stored_as(x[0], dtype, heads, dim), stored_as(x[1], dtype, heads, dim)

    def same(h):
        k, v = (torch.empty(sum(lens), heads * dim, device="cuda") for _ in range(2))
        h.gather_kv(range(3), [0] * 3, lens, k, v, ct.CT_KV_F32)
        torch.cuda.synchronize()
        assert torch.equal(k, wk) and torch.equal(v, wv)
        check_bounds(h, heads, dim, page, dtype)
        q = torch.randn(3, hq, dim, generator=g, device="cuda").bfloat16()
        plan = ct.GqaPlan(h.layout, 3, hq)
        out, sel = (torch.empty(3, hq, dim, device="cuda").bfloat16() for _ in range(2))
        picked = torch.empty(3, heads, 2, dtype=torch.int32, device="cuda")
        plan.decode(q, h.pool, h.scales, h.block_table_dev, h.seq_lens_dev, out, stream=stream())
        plan.select(q, h.bounds, h.bound_scales, h.block_table_dev, h.seq_lens_dev, picked, 2, 1, 0, stream=stream())
        plan.decode_selected(q, h.pool, h.scales, h.block_table_dev, h.seq_lens_dev, picked, 2, sel, stream=stream())
        torch.cuda.synchronize()
        NP, tb = h.layout.n_pages, torch.from_numpy(h.block_table()).cuda()
        shape = (NP, 2, heads, page, dim)
        pool = dev_copy(h.pool, shape, {BF16: torch.bfloat16, INT8: torch.int8, E4M3: torch.uint8}[dtype])
        scales = None if dtype == BF16 else dev_copy(h.scales, shape[:4], torch.float32)
        bounds = dev_copy(h.bounds, (NP, heads, 2, dim), torch.int8).cpu().numpy()
        bs = dev_copy(h.bound_scales, (NP, heads), torch.float32).cpu().numpy()
        want = G.select(q.float().cpu().numpy(), bounds, bs, tb.cpu().numpy(), lens, NP, page, hq, MOD, 2, 1, 0)
        assert np.array_equal(picked.cpu().numpy(), want)
        G.check_attention(out, None, G.attend(q, pool, scales, tb, lens, dtype, hq, MOD), dim, max(lens), dtype)
        G.check_attention(sel, None, G.attend(q, pool, scales, tb, lens, dtype, hq, MOD, pages=want), dim, max(lens), dtype)

    same(kv)
    kv.compact()
    assert sorted(kv.block_table()[kv.block_table() >= 0].tolist()) == list(range(7))
    same(kv)
    kv.save(tmp_path / "p.bin")
    back = ct.GqaKV.load(tmp_path / "p.bin", stream=stream())
    same(back)
    back.compact()
    same(back)


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_one_append_that_uses_pages_again_keeps_the_last_tokens(dtype):
    """A call longer than the window frees pages and takes them again: a slot is written by its last token alone, K and V, codes
    and scales."""
    heads, dim, page, window = 3, 64, 16, 40
    g = gen(93)
    kv = ct.GqaKV(2, 64, 9, heads, dim, page, window_tokens=window, dtype=dtype, keep_bounds=True, stream=stream())
    n = [700, 333]
    x = rows(sum(n), heads, dim, g)
    kv.append_kv([0, 1], n, x[0], x[1])
    kept = [c - (c - window) // page * page for c in n]               # tokens of the pages that the window reaches
    k, v = (torch.empty(sum(kept), heads * dim, device="cuda") for _ in range(2))
    kv.gather_kv([0, 1], [c - m for c, m in zip(n, kept)], kept, k, v, ct.CT_KV_F32)
    torch.cuda.synchronize()
    for got, src in ((k, x[0]), (v, x[1])):
        want = torch.cat((src[n[0] - kept[0]:n[0]], src[n[0] + n[1] - kept[1]:]))
        assert torch.equal(got, stored_as(want, dtype, heads, dim))
    check_bounds(kv, heads, dim, page, dtype)


# ---- what page bounds and scores are for ---------------------------------------------------------------------------------

def rounded_queries(q):
    """Whole-number codes of query heads [..., dim] and their steps, single 32-bit roundings; in 64 bits."""
    x = q.float()
    e = x.abs().amax(-1) / torch.full_like(x[..., 0], 127.0)
    c = torch.where(e[..., None] > 0, torch.round(x / e[..., None]), torch.zeros_like(x)).clamp(-127, 127)
    return c.double(), e.double()


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
@pytest.mark.parametrize("dim,page,group", [(32, 16, 1), (96, 48, 3), (128, 64, 4), (256, 128, 17)])
def test_a_page_scores_no_less_than_any_of_its_keys(dim, page, group, dtype):
    """The score of a page, from its stored bounds, against the product of the rounded query with every key of the page, and the
    pages left out against those chosen.

    s and y = b / s are single roundings, and codes are clamped only where |b| is the page's largest value, so a bound times s
    falls short of its b by at most (2^-24 + 2^-24) times that largest value `top`, and a product of `dim` terms by that times
    sum |c| e; twice as much is allowed.  The kernel's score rounds twice more: 2^-23 of it, twice that allowed."""
    g = gen(dim + group + dtype)
    heads, n_pages, pick = 2, 40, 9
    hq, width = heads * group, heads * dim
    layout = ct.GqaLayout(heads, dim, page, dtype, n_pages, n_pages)
    pool, scales = G.make_pool(n_pages, heads, page, dim, dtype, g)
    n = n_pages * page - 5
    x = torch.randn(n, 2 * width, generator=g, device="cuda")
    x[:, :width] = x[:, :width] * (torch.rand(width, generator=g, device="cuda") * 3 + 0.1) + torch.randn(width, generator=g, device="cuda")
    x[torch.rand(n, generator=g, device="cuda") < 0.02] *= 20.0
    x = x.bfloat16()
    table = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).view(1, n_pages)
    t = torch.arange(n, device="cuda")
    slots = (table[0, t // page] * page + t % page).to(torch.int32)
    ct.gqa_write_slots(layout, pool, scales, x, x[:, width:], slots, n, k_stride=2 * width, v_stride=2 * width, stream=stream())
    bounds = torch.zeros(n_pages, heads, 2, dim, dtype=torch.int8, device="cuda")
    bs = torch.zeros(n_pages, heads, device="cuda")
    counts = torch.full((n_pages,), page, dtype=torch.int32, device="cuda")
    counts[-1] = page - 5
    ct.gqa_page_bounds(layout, pool, scales, table, counts, n_pages, bounds, bs, stream=stream())
    q = torch.randn(1, hq, dim, generator=g, device="cuda").bfloat16()
    plan = ct.GqaPlan(layout, 1, hq, head_order=BLK)
    picked = torch.zeros(1, heads, pick, dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    plan.select(q, bounds, bs, table, lens, picked, pick, 1, 1, stream=stream())
    torch.cuda.synchronize()
    code, e = rounded_queries(q.view(heads, group, dim))
    for h in range(heads):
        at = table[0].long()
        keys = G.values(pool[at, 0, h], None if scales is None else scales[at, 0, h], dtype)          # [page][slot][dim]
        live = (torch.arange(page, device="cuda")[None] < counts[:, None])
        keys = torch.where(live[..., None], keys, torch.zeros_like(keys))
        product = torch.einsum("gd,ptd->gpt", code[h] * e[h][:, None], keys).masked_fill(~live[None], float("-inf"))
        hi, lo = bounds[at, h, 0].double(), bounds[at, h, 1].double()
        score = (code[h].clamp(min=0) @ hi.T + code[h].clamp(max=0) @ lo.T) * e[h][:, None] * bs[at, h].double()[None]
        top = keys.abs().amax((1, 2))
        short = 2.0 ** -22 * top[None] * (code[h].abs().sum(-1) * e[h])[:, None]
        assert (product.amax(-1) <= score + short).all()
        best = score.amax(0)
        chosen = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
        chosen[picked[0, h].long()] = True
        free = chosen.clone()
        free[0] = free[-1] = False
        assert int(chosen.sum()) == pick and bool(chosen[0]) and bool(chosen[-1])
        least = best[free].min()
        assert (best[~chosen] <= least + 2.0 ** -22 * best.abs().max()).all()
        limit = least + 2.0 ** -22 * best.abs().max() + short.amax(0)[~chosen]
        assert (product.amax(-1).amax(0)[~chosen] <= limit).all()


@pytest.mark.parametrize("dtype", [BF16, INT8, E4M3])
def test_chosen_pages_hold_the_weight(dtype):
    """Three keys a query head point along it, in pages anywhere; the other 3188 are short.  With logits of 3 |q|^2 / sqrt(128)
    (at least 18 where |q|^2 >= 68, five deviations below its mean) against others whose exponentials sum to less than 2^13,
    the pages left out hold less than 2^13 e^-18 < 2^-12 of the softmax; the decode over the chosen ones then differs from the
    whole by at most twice that of the values, besides each one's own rounding."""
    g = gen(95)
    heads, group, dim, page, n_pages, pick = 2, 4, 128, 16, 200, 16
    hq, width, n = heads * group, heads * dim, 200 * 16
    q = torch.randn(1, hq, dim, generator=g, device="cuda").bfloat16()
    assert float(q.float().square().sum(-1).min()) >= 68
    x = torch.randn(2, n, heads, dim, generator=g, device="cuda") * 0.3
    where = torch.randperm(n, generator=g, device="cuda")[:3 * group * heads].view(heads, group, 3)
    for h in range(heads):
        for i in range(group):
            x[0, where[h, i], h] = 3.0 * q[0, i * heads + h].float()
    x = x.view(2, n, width).bfloat16()
    kv = ct.GqaKV(1, n_pages, n_pages, heads, dim, page, dtype=dtype, keep_bounds=True, stream=stream())
    kv.set_free_order(np.random.default_rng(8).permutation(n_pages))
    kv.append_kv([0], [n], x[0], x[1])
    plan = ct.GqaPlan(kv.layout, 1, hq)
    picked = torch.zeros(1, heads, pick, dtype=torch.int32, device="cuda")
    out, sel = (torch.empty(1, hq, dim, device="cuda").bfloat16() for _ in range(2))
    plan.select(q, kv.bounds, kv.bound_scales, kv.block_table_dev, kv.seq_lens_dev, picked, pick, stream=stream())
    plan.decode(q, kv.pool, kv.scales, kv.block_table_dev, kv.seq_lens_dev, out, stream=stream())
    plan.decode_selected(q, kv.pool, kv.scales, kv.block_table_dev, kv.seq_lens_dev, picked, pick, sel, stream=stream())
    k = torch.empty(2, n, width, device="cuda")
    kv.gather_kv([0], [0], [n], k[0], k[1], ct.CT_KV_F32)
    torch.cuda.synchronize()
    k = k.double().view(2, n, heads, dim)
    for h in range(heads):
        pages = picked[0, h].long()
        assert set((where[h] // page).flatten().tolist()) <= set(pages.tolist())
        held = torch.isin(torch.arange(n, device="cuda") // page, pages)
        for i in range(group):
            p = torch.softmax(k[0, :, h] @ q[0, i * heads + h].double() / dim ** 0.5, 0)
            assert float(p[~held].sum()) <= 2.0 ** -12
    gap = (out.double() - sel.double()).abs()
    assert (gap <= 2 * 2.0 ** -12 * k[1].abs().max() + 3 * 2.0 ** -8 * out.double().abs().clamp(min=2.0 ** -4)).all()
