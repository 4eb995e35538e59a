"""The paged-cache operators on the GPU at the edges of what their callers may pass."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import RANGE, TYPES, Meta, Pool, attend, check_attention, check_on_gpu, dev, host, make, row_bound, tables, tt
from test_gpu_paged import torch as torch  # the fixture

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- windows
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 64, 2**30])
@pytest.mark.parametrize("new,total", [([4, 1], [1, 30]), ([3, 2], [1, 0]), ([100], [60]), ([140], [3]), ([1, 90, 5], [9, 40, 5])])
def test_windows_wider_than_any_sequence(pkg, torch, t, kv, window, new, total):
    """No limit, given as a large window: as window 0, also with more new rows than positions."""
    rng = np.random.default_rng(sum(new) + sum(total))
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "slot", 4, 2, 64)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    check_attention(b, got, gl, q, pages, t, kv, 0.125, 0)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("page,layout,d", [(1, "slot", 64), (7, "head", 128), (8, "slot", 128), (16, "head", 128), (24, "slot", 64),
                                           (64, "slot", 128), (128, "head", 64)])
@pytest.mark.parametrize("new,total,window", [([1, 1, 1], [700, 331, 20], 100), ([3, 2], [515, 260], 33), ([70, 40], [700, 415], 70),
                                              ([1, 90, 2, 1], [400, 777, 90, 300], 129)])
def test_pages_released_behind_the_window(pkg, torch, t, kv, page, layout, d, new, total, window):
    """Table entries before the first position that a sequence's new rows attend to name no page."""
    rng = np.random.default_rng(page + len(new))
    b, q, pages, pool = make(torch, rng, t, kv, new, total, page, layout, 4, 2, d)
    live = b.table.copy()
    dead = 0
    for s in range(b.seqs):
        gone = max(0, total[s] - new[s] + 1 - window) // page
        b.table[s, :gone] = np.resize([-1, b.pages, 2**31 - 1, -2**31], gone)
        dead += gone
    assert dead
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    b.table = live
    check_attention(b, got, gl, q, pages, t, kv, d ** -0.5, window)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new", [[1], [2], [300]])
def test_released_pages_of_long_caches(pkg, torch, t, kv, new):
    """The same where the work is split over the positions; a bad page that a row does attend to still counts."""
    g = torch.Generator(device="cuda").manual_seed(1)
    L, window, page = 6000, 2500, 16
    b = ref.Batch(np.random.default_rng(2), new, [L], page)
    pool = Pool(torch, kv, b, 2, 128, "slot")
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    q = ref.round_to(np.random.default_rng(3).standard_normal((b.rows, 4, 128)), t)
    live, first = b.table.copy(), max(0, L - new[0] + 1 - window)
    b.table[0, :first // page] = -1
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    bad = b.table.copy()
    b.table = live
    check_on_gpu(torch, b, got, gl, q, pool, t, kv, window)
    bad[0, first // page] = -1
    b.table = bad
    assert attend(pkg, torch, b, q, pool, t, window=window)[2] == RANGE


# ---------------------------------------------------------------- rows that are computed again
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,hq,hk", [([1500], [1500], 8, 4), ([300] * 6, [1300 - 70 * s for s in range(6)], 16, 4), ([50], [2900], 8, 2)])
def test_rows_that_are_computed_again_among_others(pkg, torch, t, kv, new, total, hq, hk):
    """An infinite value early in one head of each sequence: all of the head's rows are computed
    again, several items per CTA (and split ones); element 7 is infinite, everything else as ever."""
    b = ref.Batch(np.random.default_rng(1), new, total, 16)
    g = torch.Generator(device="cuda").manual_seed(5)
    pool = Pool(torch, kv, b, hk, 64, "slot")
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    q = ref.round_to(np.random.default_rng(2).standard_normal((b.rows, hq, 64)) * 1.5, t)
    at = [b.place(s, 5) for s in range(b.seqs)]
    for pg, sl in at:
        pool.t[1][pg, sl, 1, 7] = np.inf
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    assert st == 0
    reach = np.zeros((b.rows, hq), bool)
    for s in range(b.seqs):
        for i in range(new[s]):
            reach[b.start[s] + i, hq // hk:2 * hq // hk] = total[s] - new[s] + i >= 5
    assert np.isposinf(got[reach][:, 7]).all() and np.isfinite(got[~reach]).all()
    for pg, sl in at:
        pool.t[1][pg, sl, 1, 7] = 0.0
    clean, _, _ = attend(pkg, torch, b, q, pool, t)
    got[..., 7] = np.where(reach, clean[..., 7], got[..., 7])
    check_on_gpu(torch, b, got, gl, q, pool, t, kv)


@pytest.mark.parametrize("new,total", [([1100], [1100]), ([40], [4500])])
@pytest.mark.parametrize("which", [0, 1])
def test_f32_rows_of_unlike_size_in_one_tile(pkg, torch, new, total, which):
    """A row of K (V) 1e-6 times its neighbours': its tile's rows are computed again."""
    b = ref.Batch(np.random.default_rng(1), new, total, 16)
    g = torch.Generator(device="cuda").manual_seed(6)
    pool = Pool(torch, "f32", b, 2, 128, "head")
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    pg, sl = b.place(0, 100)
    pool.t[which][pg, :, sl] *= 1e-6
    q = ref.round_to(np.random.default_rng(2).standard_normal((b.rows, 4, 128)) * 1.5, "f32")
    got, gl, st = attend(pkg, torch, b, q, pool, "f32")
    assert st == 0
    check_on_gpu(torch, b, got, gl, q, pool, "f32", "f32")


def test_rows_computed_again_where_a_cta_has_many_items(pkg, torch):
    """76,800 items, some 519 per CTA: the marks of the first and the last share a place."""
    seqs, n, heads, d = 1200, 17, 64, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (torch.randn(seqs, n, heads, d, generator=g, device="cuda").half() for _ in range(3))
    hit = torch.tensor([0, 1, 600, seqs - 2, seqs - 1], device="cuda")
    v[hit, 3, 7, 9] = float("inf")
    out = torch.full_like(q, -7.0)
    lse = torch.full((seqs * n, heads), -7.0, device="cuda")
    start = torch.arange(0, seqs * n + 1, n, dtype=torch.int32, device="cuda")
    length = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    table = torch.arange(seqs, dtype=torch.int32, device="cuda")
    work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.engine.paged_attention(q.data_ptr(), out.data_ptr(), seqs * n, heads, heads, d, k.data_ptr(), v.data_ptr(), seqs, n,
                               start.data_ptr(), length.data_ptr(), table.data_ptr(), 1, seqs, n, work.data_ptr(),
                               lse_ptr=lse.data_ptr(), dtype="f16", kv_dtype="f16", page_strides=(n * heads * d, d, heads * d),
                               status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    reach = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    reach[hit, 3:, 7, 9] = True
    assert torch.equal(torch.isposinf(out), reach) and not torch.isnan(out).any()
    hide = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    b = ref.Batch(np.random.default_rng(0), [n], [n], n)
    v[hit, 3, 7, 9] = 0.0
    for s in range(0, seqs, 100):
        q64, k64, v64 = (z[s:s + 100].double() for z in (q, k, v))
        x = (torch.einsum("sihd,sjhd->shij", q64, k64) * d ** -0.5).masked_fill(hide, -torch.inf)
        w = torch.softmax(x, -1)
        want, mass = (torch.einsum("shij,sjhd->sihd", w, z) for z in (v64, v64.abs()))
        size = (torch.einsum("sihd,sjhd->shij", q64.abs(), k64.abs()) * d ** -0.5).masked_fill(hide, 0).amax(-1).transpose(1, 2)
        bound, lb = ref.attention_bounds(b, want.cpu().numpy(), mass.cpu().numpy(), size.cpu().numpy(), "f16", "f16", d)
        got = torch.where(reach[s:s + 100], want, out[s:s + 100].double())
        assert np.all((got - want).abs().cpu().numpy() <= bound)
        wl = torch.logsumexp(x, -1).transpose(1, 2).cpu().numpy()
        assert np.all(np.abs(host(lse.view(seqs, n, heads)[s:s + 100]) - wl) <= lb + 2.0**-23 * np.abs(wl))


def test_more_row_tiles_than_32_bits_count(pkg, torch):
    """Overlapping ranges of 2^24 rows whose tiles add up past 2^31 and 2^32: refused, nothing written."""
    rows, d = 1 << 24, 64
    q = torch.zeros(rows, d, dtype=torch.float16, device="cuda")
    out = torch.full((rows, d), -7.0, dtype=torch.float16, device="cuda")
    page = torch.zeros(2, 16, d, dtype=torch.float16, device="cuda")
    work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    for seqs in (1 << 16, 1 << 17, (1 << 17) + 64, 1 << 20):  # half of them own every row: 2^16 tiles each
        start = torch.tensor([0, rows], dtype=torch.int32, device="cuda").repeat(seqs // 2 + 1)[:seqs + 1].contiguous()
        length = torch.full((seqs,), 16, dtype=torch.int32, device="cuda")
        table = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        pkg.engine.paged_attention(q.data_ptr(), out.data_ptr(), rows, 1, 1, d, page[0].data_ptr(), page[1].data_ptr(), 1, 16,
                                   start.data_ptr(), length.data_ptr(), table.data_ptr(), 1, seqs, rows, work.data_ptr(),
                                   dtype="f16", kv_dtype="f16", status_ptr=st.data_ptr())
        torch.cuda.synchronize()
        assert int(st.item()) == RANGE
        assert bool((out == -7.0).all())


# ---------------------------------------------------------------- the largest batches
def test_as_many_single_tokens_as_there_are(pkg, torch):
    """66,000 sequences of one token over 32 kv heads, one position each: the row is its value."""
    seqs, heads, d = 66000, 32, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q, out = (torch.randn(seqs, heads * d, generator=g, device="cuda").half() for _ in range(2))
    kp, vp = (torch.randn(64, heads, 1, d, generator=g, device="cuda").half() for _ in range(2))
    start = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    length = torch.ones(seqs, dtype=torch.int32, device="cuda")
    table = (start[:seqs] % 64).contiguous()
    work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.engine.paged_attention(q.data_ptr(), out.data_ptr(), seqs, heads, heads, d, kp.data_ptr(), vp.data_ptr(), 64, 1,
                               start.data_ptr(), length.data_ptr(), table.data_ptr(), 1, seqs, 1, work.data_ptr(),
                               dtype="f16", kv_dtype="f16", status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    assert torch.equal(out.view(seqs, heads, d), vp[:, :, 0][table.long()])


@pytest.mark.parametrize("t,kv", TYPES)
def test_more_work_than_is_counted_is_out_of_range(pkg, torch, t, kv):
    """2^30 positions of single tokens: the documented status, nothing computed."""
    page = 1 << 20
    b = ref.Batch(np.random.default_rng(0), [1, 1], [page, 100], page, spare=0)
    b.pages = 1
    pool = Pool(torch, kv, b, 1, 64, "slot")
    b.len[0] = 1 << 30
    b.table, b.wide = np.zeros((2, 1024), np.int32), 1024
    q = np.ones((2, 4, 64))
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    assert st == RANGE and np.all(got == -7.0) and np.all(gl == -7.0)


@pytest.mark.parametrize("t,kv", TYPES)
def test_append_of_a_sequence_that_does_not_fit(pkg, torch, t, kv):
    """A length beyond the table row: nothing of the sequence is appended, not its fitting rows either."""
    rng = np.random.default_rng(1)
    b = ref.Batch(rng, [2, 3, 1], [8, 8, 5], 4, wide=2)
    x = ref.round_to(rng.standard_normal((b.rows, 4, 64)), t)
    before = [ref.round_to(rng.standard_normal((b.pages, 4, 1, 64)), kv) for _ in range(2)]
    pool, m = Pool(torch, kv, b, 1, 64, "slot", before), Meta(torch, b)
    m.len[1] = 9
    buf = dev(torch, x.reshape(b.rows, -1)).to(tt(torch, t))
    qo, st = torch.full((b.rows, 128), -7.0, dtype=buf.dtype, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    at, e = buf.data_ptr(), buf.element_size()
    pkg.engine.paged_append(at + 128 * e, at + 192 * e, b.rows, 1, 64, **pool.args(), **m.kw, q_ptr=at, q_out_ptr=qo.data_ptr(),
                            q_heads=2, dtype=t, q_stride=256, k_stride=256, v_stride=256, status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == RANGE
    want = [z.copy() for z in before]
    for s, p, row in ((0, 6, 0), (0, 7, 1), (2, 4, 5)):
        for z, h in zip(want, (2, 3)):
            z[b.place(s, p)] = ref.round_to(x[row, h], kv)
    assert all(np.array_equal(u, w) for u, w in zip(pool.values(), want))
    got = host(qo)
    assert np.all(got[2:5] == -7.0) and np.array_equal(got[[0, 1, 5]], x[[0, 1, 5], :2].reshape(3, -1))


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 2, 40, 300])
def test_positions_up_to_two_to_the_31(pkg, torch, t, kv, n):
    """The longest sequence a table can describe (one page, named again and again), by a window."""
    page, wide, window = 42966, 49981, 100
    L = page * wide
    assert 2**31 - 128 < L < 2**31
    rng = np.random.default_rng(n)
    b = ref.Batch(rng, [n], [page], page, spare=0)
    q = ref.round_to(rng.standard_normal((b.rows, 2, 64)), t)
    pages = [ref.round_to(rng.standard_normal((1, page, 1, 64)), kv) for _ in range(2)]
    pool = Pool(torch, kv, b, 1, 64, "slot", pages)
    b.len[:] = L
    b.table, b.wide = np.zeros((1, wide), np.int32), wide
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    b.len[:] = page  # the last positions lie in the page's last slots either way
    check_attention(b, got, gl, q, pages, t, kv, 0.125, window)


# ---------------------------------------------------------------- infinite keys
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,hq", [([1], [300], 4), ([2, 1], [90, 700], 2), ([3], [70], 4), ([64], [200], 4)])
def test_a_score_of_minus_infinity_has_no_weight(pkg, torch, t, kv, new, total, hq):
    """An infinite key whose scores are -inf: its position has no weight, the row is finite. Where
    one score is +inf, and where one is inf - inf, the row is NaN."""
    rng = np.random.default_rng(15)
    b, q, pages, _ = make(torch, rng, t, kv, new, total, 16, "head", hq, 1, 64, qmul=0.5)
    q[:, :, 3] = ref.round_to(0.3 + np.abs(q[:, :, 3]), t)
    q[:, :, 11] = ref.round_to(-0.7 - np.abs(q[:, :, 11]), t)
    at = [b.place(s, p) for s in range(b.seqs) for p in (total[s] // 3, total[s] - new[s])]
    for i, (pg, sl) in enumerate(at):
        pages[0][pg, sl, 0, 3 if i % 2 else 11] = -np.inf if i % 2 else np.inf  # scores of -inf for every row
    got, gl, st = attend(pkg, torch, b, q, Pool(torch, kv, b, 1, 64, "head", pages), t)
    assert st == 0
    hidden = [pages[0].copy(), pages[1]]
    for pg, sl in at:
        hidden[0][pg, sl, 0] = 0.0
    size = ref.attention(b, q, *hidden, 0.125, 0)[3]  # of the positions that count
    with np.errstate(invalid="ignore"):
        out, wl, mass, _ = ref.attention(b, q, *pages, 0.125, 0)
    bound, lb = ref.attention_bounds(b, out, mass, size, t, kv, 64)
    rows = int(b.start[-1])
    assert np.isfinite(out[:rows]).all()
    assert np.all(np.abs(got - out)[:rows] <= bound[:rows])
    assert np.all(np.abs(gl - wl)[:rows] <= (lb + 2.0**-23 * np.abs(wl))[:rows])
    pg, sl = at[1]
    for key in ([(3, np.inf)], [(3, np.inf), (11, np.inf)]):  # +inf; inf - inf
        two = pages[0].copy()
        for d, v in key:
            two[pg, sl, 0, d] = v
        got, gl, st = attend(pkg, torch, b, q, Pool(torch, kv, b, 1, 64, "head", [two, pages[1]]), t)
        last = slice(0, b.new[0])  # every new row of sequence 0 sees it
        assert np.isnan(got[last]).all() and np.isnan(gl[last]).all()
        other = slice(b.new[0], rows)
        assert np.all(np.abs(got - out)[other] <= bound[other])


# ---------------------------------------------------------------- append: what is left alone
def append_call(pkg, torch, b, x, pool, m, hq, hk, rope=None, t="f32"):
    """x [rows][hq + 2 hk][d]; q goes through to rows of -7. Returns q's rows and the status."""
    d = x.shape[2]
    buf = dev(torch, x.reshape(b.rows, -1)).to(tt(torch, t))
    qo, st = torch.full((b.rows, hq * d), -7.0, dtype=buf.dtype, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    at, e, w = buf.data_ptr(), buf.element_size(), buf.shape[1]
    kw = {} if rope is None else dict(cos_ptr=rope[0].data_ptr(), sin_ptr=rope[1].data_ptr(), rope_rows=rope[0].shape[0],
                                      rope_half_dim=rope[0].shape[1])
    pkg.engine.paged_append(at + hq * d * e, at + (hq + hk) * d * e, b.rows, hk, d, **pool.args(), **m.kw, q_ptr=at,
                            q_out_ptr=qo.data_ptr(), q_heads=hq, dtype=t, q_stride=w, k_stride=w, v_stride=w,
                            status_ptr=st.data_ptr(), **kw)
    torch.cuda.synchronize()
    return host(qo).reshape(b.rows, hq, d), int(st.item())


@pytest.mark.parametrize("start,kept", [
    ([-2, 1, 2, 3, 4, 5, 6, 7, 100], [1, 2, 3, 4, 5, 6]),      # the first and the last range lie outside the rows
    ([0, 1, 2, 3, 4, 5, 6, 7, 9], [0, 1, 2, 3, 4, 5, 6]),
    ([3, 4, 5, 5, 5, 5, 5, 6, 7], [3, 4, 5, 6]),               # rows before the first and behind the last sequence
    ([-2, 1, 2, 9, 1, 0, 6, 7, 100], None)])                   # in no order: nothing outside the sequences' places
def test_append_of_bad_row_ranges_leaves_the_pool_alone(pkg, torch, start, kept):
    rng = np.random.default_rng(3)
    b = ref.Batch(rng, [1] * 8, [4, 3, 4, 2, 1, 4, 4, 4], 4, wide=2)
    x = rng.standard_normal((8, 4, 64)).astype(np.float32)
    before = [rng.standard_normal((b.pages, 4, 1, 64)).astype(np.float32) for _ in range(2)]
    pool, m = Pool(torch, "f32", b, 1, 64, "slot", before), Meta(torch, b)
    m.start.copy_(dev(torch, np.array(start, np.int32)))
    got, st = append_call(pkg, torch, b, x, pool, m, 2, 1)
    assert st == (RANGE if start[0] < 0 or start[-1] > 8 else 0)
    if kept is None:  # every place that differs is that of a sequence's newest positions
        own = np.zeros(before[0].shape[:2], bool)
        for s in range(8):
            for p in range(b.total[s]):
                own[b.place(s, p)] = True
        assert all(np.array_equal(u[~own], w[~own]) for u, w in zip(pool.values(), before))
        return
    want = [z.copy() for z in before]
    for row in kept:
        s = max(i for i in range(8) if start[i] <= row)
        for z, h in zip(want, (2, 3)):
            z[b.place(s, b.total[s] - 1)] = x[row, h]
    assert all(np.array_equal(u, w) for u, w in zip(pool.values(), want))
    gone = [r for r in range(8) if r not in kept]
    assert np.array_equal(got[kept], x[kept, :2]) and np.all(got[gone] == -7.0)


@pytest.mark.parametrize("t,kv", TYPES)
def test_append_behind_the_rotation_tables(pkg, torch, t, kv):
    """Positions that the tables do not reach: k, v and q of those rows stay as they were."""
    rng = np.random.default_rng(4)
    b = ref.Batch(rng, [5, 1, 2], [12, 10, 3], 4)
    top, hq, hk, d = 10, 3, 2, 64
    x = ref.round_to(rng.standard_normal((b.rows, hq + 2 * hk, d)), t)
    before = [ref.round_to(rng.standard_normal((b.pages, 4, hk, d)), kv) for _ in range(2)]
    cos, sin = tables(rng, top, 32)
    pool, m = Pool(torch, kv, b, hk, d, "head", before), Meta(torch, b)
    got, st = append_call(pkg, torch, b, x, pool, m, hq, hk, rope=(dev(torch, cos), dev(torch, sin)), t=t)
    assert st == RANGE
    want, near = [z.copy() for z in before], np.zeros_like(before[0])
    for s in range(b.seqs):
        for i in range(b.new[s]):
            p, row = b.total[s] - b.new[s] + i, b.start[s] + i
            if p >= top:
                assert np.all(got[row] == -7.0)
                continue
            val, mag = ref.norm_rope(x[row:row + 1, :hq + hk], None, 0, cos[p:p + 1], sin[p:p + 1])
            assert np.all(np.abs(got[row] - val[0, :hq]) <= row_bound(val, mag, t)[0, :hq])
            at = b.place(s, p)
            want[0][at], near[at] = val[0, hq:], row_bound(val, mag, kv)[0, hq:]
            want[1][at] = ref.round_to(x[row, hq + hk:], kv)
    kp, vp = pool.values()
    assert np.array_equal(vp, want[1]) and np.all(np.abs(kp - want[0]) <= near)


@pytest.mark.parametrize("t,kv", TYPES)
def test_append_to_a_page_that_does_not_exist_turns_q(pkg, torch, t, kv):
    rng = np.random.default_rng(5)
    b = ref.Batch(rng, [2, 1], [6, 3], 4)
    x = ref.round_to(rng.standard_normal((b.rows, 3, 64)), t)
    before = [ref.round_to(rng.standard_normal((b.pages, 4, 1, 64)), kv) for _ in range(2)]
    want = [z.copy() for z in before]
    for z, h in zip(want, (1, 2)):
        z[b.place(1, 2)] = ref.round_to(x[2, h], kv)
    b.table[0, 1] = b.pages
    pool, m = Pool(torch, kv, b, 1, 64, "slot", before), Meta(torch, b)
    got, st = append_call(pkg, torch, b, x, pool, m, 1, 1, t=t)
    assert st == RANGE and np.array_equal(got[:, 0], x[:, 0])
    assert all(np.array_equal(u, w) for u, w in zip(pool.values(), want))


# ---------------------------------------------------------------- strides
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("page,layout,d", [(8, "slot", 64), (16, "head", 128), (16, "slot", 128), (64, "head", 64), (128, "slot", 128),
                                           (128, "head", 64), (256, "head", 128)])
@pytest.mark.parametrize("gap", [8, 64])
@pytest.mark.parametrize("new,total,window", [([200, 90], [700, 333], 0), ([130, 1, 3], [130, 300, 515], 150)])
def test_pages_with_gaps(pkg, torch, t, kv, page, layout, d, gap, new, total, window):
    """NaN between the rows of the pages (TMA boxes of padded slots, heads and pages)."""
    rng = np.random.default_rng(page + gap)
    b, q, pages, pool = make(torch, rng, t, kv, new, total, page, layout, 4, 2, d, gap=gap)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window, pad=8, qpad=24)
    assert st == 0
    for z, p in zip(pool.t, pages):
        p = p if layout == "slot" else p.transpose(0, 2, 1, 3)
        z[..., :d] = dev(torch, np.nan_to_num(p, nan=0.0, posinf=0.0)).to(z.dtype)  # stale slots, for the 64-bit form
    check_on_gpu(torch, b, got, gl, q, pool, t, kv, window)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 150])
def test_k_and_v_interleaved_in_one_pool(pkg, torch, t, kv, n):
    """[page][K, V][slot][head][d], pages twice as far apart as they are long."""
    page, hk, d = 16, 2, 64
    rng = np.random.default_rng(n)
    b = ref.Batch(rng, [n, n], [400, 220], page)
    both = torch.randn(b.pages, 2, page, hk, d, device="cuda").to(tt(torch, kv))
    pool = Pool.__new__(Pool)
    pool.torch, pool.kv, pool.b, pool.hk, pool.d, pool.layout = torch, kv, b, hk, d, "slot"
    pool.t, pool.strides = [both[:, 0], both[:, 1]], (2 * page * hk * d, d, hk * d)
    q = ref.round_to(rng.standard_normal((b.rows, 6, d)), t)
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    assert st == 0
    check_on_gpu(torch, b, got, gl, q, pool, t, kv)


# ---------------------------------------------------------------- log-sum-exp
def lse_bound(wl, size, longest, dim):
    """lse is made of unrounded f32 weights: an error ds of each score (attention_bounds) with the
    exponential's own, the f32 sum over the positions (2^-23 each), log2 (2^-22) and its two
    roundings with the sum's logarithm and the maximum, up to |lse| + 16 (2^-23 of it)."""
    ds = (dim * 2.0**-23 + 2.0**-21) * size + 2.0**-20
    return ds + longest * 2.0**-23 + 2.0**-22 + 2.0**-23 * (np.abs(wl) + 16)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,window", [([1, 1, 1], [2, 700, 63], 0), ([3, 2], [300, 40], 25), ([90, 40], [300, 41], 0), ([140], [420], 64)])
def test_log_sum_exp_counts_unrounded_weights(pkg, torch, t, kv, new, total, window):
    rng = np.random.default_rng(sum(total))
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "head", 4, 2, 64, extra=0)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    _, wl, _, size = ref.attention(b, q, *pages, 0.125, window)
    assert st == 0 and np.all(np.abs(gl - wl) <= lse_bound(wl, size, max(total), 64))


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 100])
def test_log_sum_exp_of_equal_scores(pkg, torch, t, kv, n):
    """Weights that a 16-bit type cannot hold: with scores of 0 and one of ln 1.0039 (q = 0 but
    for one element), the sum is known, and a rounded weight would show."""
    rng = np.random.default_rng(1)
    b, q, pages, pool = make(torch, rng, t, kv, [n], [260], 16, "slot", 2, 1, 64, extra=0)
    q[:] = 0.0
    q[:, :, 0] = 1.0
    for p in range(260):
        pages[0][b.place(0, p)] = 0.0
        pages[0][b.place(0, p) + (0, 0)] = ref.round_to(0.0039 * (p % 7), kv)
    pool = Pool(torch, kv, b, 1, 64, "slot", pages)
    got, gl, st = attend(pkg, torch, b, q, pool, t, scale=1.0)
    _, wl, _, size = ref.attention(b, q, *pages, 1.0, 0)
    # one product per score, exact: the scores' error is that of the exponential alone
    assert st == 0 and np.all(np.abs(gl - wl) <= 2.0**-20 + 260 * 2.0**-23 + 2.0**-22 + 2.0**-23 * (np.abs(wl) + 16))


# ---------------------------------------------------------------- the weights' bits
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total", [([1, 1, 1], [2, 90, 40]), ([2, 1], [60, 7]), ([30, 40], [30, 60])])
def test_weights_are_as_exact_as_they_are_said_to_be(pkg, torch, t, kv, new, total):
    """q = 0 but for one element, so that the scores are exact: what is left is the weights' own
    error, 22 bits (bf16: 16) for few rows and f32 rows, half a step of the type for chunks."""
    rng = np.random.default_rng(3)
    b, q, pages, _ = make(torch, rng, t, kv, new, total, 16, "slot", 2, 1, 64, extra=0)
    q[:, :, 1:] = 0.0
    pages[0] = np.nan_to_num(pages[0], nan=0.0, posinf=0.0)
    pages[0][..., 1:] = 0.0
    got, gl, st = attend(pkg, torch, b, q, Pool(torch, kv, b, 1, 64, "slot", pages), t, scale=1.0)
    out, _, mass, size = ref.attention(b, q, *pages, 1.0, 0)
    weight = 2.0**-21 if t == "f32" else {"f16": 2.0**-21, "bf16": 2.0**-16}[t] if max(new) <= 2 else ref.HALF_STEP[t]
    ds = 2.0**-20 + 2.0**-22 * size  # an exact product, its scaling by log2(e), the exponential
    if t == "f32":
        ds = ds + 2.0**-21 * size
    rel = 2 * ds + weight + 2 * max(total) * 2.0**-23
    bound = rel[..., None] * mass * 1.01 + ref.HALF_STEP[t] * np.abs(out) * 1.01 + 2 * ref.TINY[t]
    assert st == 0 and np.all(np.abs(got - out) <= bound)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("gap", [4, 9, 14, 18])
def test_small_weights_beside_a_large_one(pkg, torch, t, kv, n, gap):
    """One position whose score lies `gap` above all others, with a value of 0: the result is made
    of small weights alone. They have their relative error, or 2^-31 of the largest weight."""
    rng = np.random.default_rng(gap)
    L = 300
    b, q, pages, _ = make(torch, rng, t, kv, [n], [L], 16, "slot", 2, 1, 64, extra=0)
    q[:] = 0.0
    q[:, :, 0] = 1.0
    pages[0] = np.zeros_like(pages[0])
    pages[1] = ref.round_to(np.abs(np.nan_to_num(pages[1], nan=0.0, posinf=0.0)) + 1.0, kv)
    pg, sl = b.place(0, 20)
    pages[0][pg, sl, 0, 0], pages[1][pg, sl] = gap, 0.0
    got, gl, st = attend(pkg, torch, b, q, Pool(torch, kv, b, 1, 64, "slot", pages), t, scale=1.0)
    out, _, mass, size = ref.attention(b, q, *pages, 1.0, 0)
    weight = {"f32": 2.0**-21, "f16": 2.0**-21 if n == 1 else 2.0**-11, "bf16": 2.0**-16 if n == 1 else 2.0**-8}[t]
    ds = 2.0**-20 + 2.0**-21 * size  # exact products, their scaling by log2(e), the exponential
    rel = 2 * ds + weight + 2 * L * 2.0**-23
    floor = 0.0 if t == "bf16" else L * 2.0**-31 * np.abs(pages[1]).max()
    bound = rel[..., None] * mass * 1.01 + floor + ref.HALF_STEP[t] * np.abs(out) * 1.01 + 2 * ref.TINY[t]
    assert st == 0 and np.all(np.abs(got - out) <= bound)


# ---------------------------------------------------------------- heads and graphs
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("hq,hk,d", [(128, 1, 64), (100, 1, 64), (7, 1, 128), (10, 2, 64), (33, 3, 64), (36, 2, 128)])
@pytest.mark.parametrize("new,total,window", [([1, 1], [90, 7], 0), ([5, 2], [40, 70], 30), ([19], [140], 0)])
def test_any_number_of_heads_per_kv_head(pkg, torch, t, kv, hq, hk, d, new, total, window):
    rng = np.random.default_rng(hq)
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "slot", hq, hk, d)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    check_attention(b, got, gl, q, pages, t, kv, d ** -0.5, window)


@pytest.mark.parametrize("t,kv", TYPES)
def test_a_captured_batch_of_tokens_and_chunks_grows(pkg, torch, t, kv):
    """Single tokens and chunks in one captured call (both kernels and their joins), replayed with
    other lengths, other row ranges and another table."""
    hq, hk, d, page, window = 8, 4, 64, 16, 900
    rng = np.random.default_rng(16)
    rounds = [[1] * 40 + [150, 90], [1] * 39 + [33, 1, 207], [0, 2] * 20 + [200, 0]]
    totals = [[n + int(rng.integers(0, 1000)) for n in new] for new in rounds]
    rows, wide, seqs = 280, 80, 42
    pages = 3000
    g = torch.Generator(device="cuda").manual_seed(3)
    first = ref.Batch(np.random.default_rng(0), rounds[0], totals[0], page, wide=wide)
    first.pages = pages
    pool = Pool(torch, kv, first, hk, d, "slot")
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    m = Meta(torch, first)
    dq = torch.zeros(rows, hq * d, dtype=tt(torch, t), device="cuda")
    out, lse = torch.empty_like(dq), torch.empty(rows, hq, device="cuda")
    work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.engine.paged_attention(dq.data_ptr(), out.data_ptr(), rows, hq, hk, d, **pool.args(), **m.kw, max_q=207,
                                   work_ptr=work.data_ptr(), window=window, lse_ptr=lse.data_ptr(), dtype=t,
                                   status_ptr=st.data_ptr(), stream=torch.cuda.current_stream())
    for new, total in zip(rounds, totals):
        b = ref.Batch(rng, new, total, page, wide=wide)
        table = rng.integers(0, pages, seqs * wide).astype(np.int32)  # pages may be shared
        b.table = table.reshape(seqs, wide)
        q = ref.round_to(rng.standard_normal((rows, hq, d)) * 1.5, t)
        dq.copy_(dev(torch, q.reshape(rows, -1)))
        for x, y in ((m.start, b.start), (m.len, b.len), (m.table, b.table)):
            x.copy_(dev(torch, y))
        out.fill_(-7.0)
        work.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert int(st.item()) == 0
        got = host(out).reshape(rows, hq, d)
        assert np.all(got[b.start[-1]:] == -7.0)
        live = [s for s in range(seqs) if new[s]]  # the 64-bit form is of sequences with rows
        b.seqs, b.new, b.total = len(live), [new[s] for s in live], [total[s] for s in live]
        b.start, b.table = np.append(b.start[live], b.start[-1]), b.table[live]
        check_on_gpu(torch, b, got, host(lse), q, pool, t, kv, window)


@pytest.mark.parametrize("n", [1, 90])
def test_small_elements_beside_large_ones_in_f32_pages(pkg, torch, n):
    """window 1: a row is its own position's value. Elements down to 2^-30 of their neighbours keep 22
    bits or come within 2^-38 of the largest |v| of the 64 positions (single tokens: 22 bits)."""
    rng = np.random.default_rng(3)
    b, q, pages, _ = make(torch, rng, "f32", "f32", [n], [300], 16, "slot", 2, 1, 64, extra=0)
    pages[1] = ref.round_to(np.nan_to_num(pages[1], nan=0.0, posinf=0.0) * 2.0 ** -rng.integers(0, 30, pages[1].shape), "f32")
    pages[1][..., 0] = 1.0  # rows of like size
    got, gl, st = attend(pkg, torch, b, q, Pool(torch, "f32", b, 1, 64, "slot", pages), "f32", window=1)
    v = np.stack([pages[1][b.place(0, p)][0] for p in range(300 - n, 300)])[:, None]
    floor = 0.0 if n == 1 else 2.0**-38 * np.abs(pages[1]).max()
    # the weight's halves, the value's halves, the product's sum and the quotient
    assert st == 0 and np.all(np.abs(got - v) <= (2.0**-21 + 2.0**-22 + 2.0**-22) * np.abs(v) + floor)
