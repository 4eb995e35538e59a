"""The paged-cache operators on the GPU (qora_qk_norm_rope, qora_paged_append,
qora_paged_attention) against their plain 64-bit forms (paged_ref.py), element by element
within bounds that count the operators' roundings."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
RANGE = 5


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def tt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def dev(torch, a, dtype=None):
    t = torch.from_numpy(np.array(a, order="C"))  # a copy that is contiguous
    return t.to("cuda") if dtype is None else t.to(dtype).to("cuda")


def host(t):
    return t.double().cpu().numpy()


class Pool:
    """Pages on the GPU in either order, with their 64-bit values as [page][slot][head][d]."""

    def __init__(self, torch, kv, b, hk, d, layout, fill=None, gap=0):
        self.torch, self.kv, self.b, self.hk, self.d, self.layout = torch, kv, b, hk, d, layout
        ps = b.page
        inner = (ps, hk) if layout == "slot" else (hk, ps)
        self.t = [torch.zeros((b.pages, *inner, d + gap), dtype=tt(torch, kv), device="cuda") for _ in range(2)]
        w = d + gap
        self.strides = (ps * hk * w, w, hk * w) if layout == "slot" else (ps * hk * w, ps * w, w)
        if fill is not None:
            for t, f in zip(self.t, fill):
                f = f if layout == "slot" else f.transpose(0, 2, 1, 3)
                t[..., :d] = dev(torch, f).to(t.dtype)
                if gap:
                    t[..., d:] = float("nan")

    def values(self):
        v = [host(t)[..., :self.d] for t in self.t]
        return [x if self.layout == "slot" else x.transpose(0, 2, 1, 3) for x in v]

    def args(self):
        return dict(k_pages_ptr=self.t[0].data_ptr(), v_pages_ptr=self.t[1].data_ptr(), num_pages=self.b.pages,
                    page_size=self.b.page, page_strides=self.strides, kv_dtype=self.kv)


class Meta:
    def __init__(self, torch, b):
        self.start, self.len, self.table = (dev(torch, x) for x in (b.start, b.len, b.table))
        self.kw = dict(q_start_ptr=self.start.data_ptr(), kv_len_ptr=self.len.data_ptr(), table_ptr=self.table.data_ptr(),
                       table_stride=b.wide, seqs=b.seqs)


def tables(rng, top, r):
    a = rng.uniform(0, 2 * np.pi, (top, r))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


# roundings of a normalised and rotated element, in units of 2^-24 of the magnitudes it is
# made of: the norm's sum (16 + 4 additions, halved by the root: 10), mean, eps, root,
# quotient and two products (6), the rotation's product and sum (2): below 24
ROW_STEPS = 24 * 2.0**-24


def row_bound(val, mag, t):
    return ROW_STEPS * mag + ref.HALF_STEP[t] * np.abs(val) * 1.001 + ref.TINY[t]


# ---------------------------------------------------------------- norm and rotation
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,hq,hk,d,r,gains,joined", [
    (1, 16, 4, 128, 64, True, True), (3, 5, 3, 64, 32, True, False), (7, 16, 4, 128, 32, False, True),
    (2, 0, 7, 64, 8, True, False), (33, 3, 0, 128, 64, True, False), (5, 4, 4, 64, 24, False, True),
    (4, 2, 1, 128, None, True, True), (1031, 16, 4, 128, 64, True, True), (700, 24, 1, 64, 16, True, True)])
def test_norm_rope(pkg, torch, t, rows, hq, hk, d, r, gains, joined):
    rng = np.random.default_rng(rows * 100 + hq)
    x = ref.round_to(rng.standard_normal((rows, hq + hk + 1, d)) * rng.uniform(0.01, 30, (rows, 1, 1)), t)
    if rows > 2:
        x[2] = 0.0  # a row of zeros: eps alone under the root
    g = [rng.uniform(-2, 2, d).astype(np.float32) if gains else None for _ in range(2)]
    top = 50
    pos = rng.integers(0, top, rows).astype(np.int32)
    if rows > 4:
        pos[3] = -1  # padding
    cos, sin = tables(rng, top, r or 8)
    buf = dev(torch, x.reshape(rows, -1)).to(tt(torch, t))
    q, k = buf[:, :hq * d], buf[:, hq * d:(hq + hk) * d]
    if not joined:
        q, k = q.contiguous(), k.contiguous()
    pad = 16
    qo, ko = (torch.full((rows, h * d + pad), -7.0, dtype=buf.dtype, device="cuda") for h in (hq, hk))
    dp, dc, ds = dev(torch, pos), dev(torch, cos), dev(torch, sin)
    dg = [None if y is None else dev(torch, y) for y in g]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    ptr = lambda z: None if z is None else z.data_ptr()  # noqa: E731
    pkg.engine.qk_norm_rope(q.data_ptr() if hq else None, k.data_ptr() if hk else None, qo.data_ptr(), ko.data_ptr(), rows,
                            hq, hk, d, ptr(dp) if r else None, ptr(dc) if r else None, ptr(ds) if r else None, top,
                            r or 0, ptr(dg[0]), ptr(dg[1]), 1e-5, dtype=t, q_stride=q.stride(0) if hq else None,
                            k_stride=k.stride(0) if hk else None, q_out_stride=hq * d + pad, k_out_stride=hk * d + pad,
                            status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    live = pos >= 0 if r else np.ones(rows, bool)
    for out, h0, h, gamma in ((qo, 0, hq, g[0]), (ko, hq, hk, g[1])):
        got = host(out)
        assert np.all(got[:, h * d:] == -7.0) and np.all(got[~live] == -7.0)
        val, mag = ref.norm_rope(x[live, h0:h0 + h], gamma, 1e-5, cos[pos[live]] if r else None, sin[pos[live]] if r else None)
        assert np.all(np.abs(got[live, :h * d].reshape(val.shape) - val) <= row_bound(val, mag, t))


def test_norm_rope_in_place_and_out_of_table(pkg, torch):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 4, 64)).astype(np.float32)
    pos = np.array([0, 9, 10, 3, 2**31 - 1, 1], np.int32)  # rows 2 and 4 lie behind the ten rows of the tables
    cos, sin = tables(rng, 10, 32)
    buf, dp, dc, ds = dev(torch, x.reshape(6, -1)), dev(torch, pos), dev(torch, cos), dev(torch, sin)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    at = buf.data_ptr()
    pkg.engine.qk_norm_rope(at, at + 2 * 64 * 4, at, at + 2 * 64 * 4, 6, 2, 2, 64, dp.data_ptr(), dc.data_ptr(),
                            ds.data_ptr(), 10, 32, q_stride=256, k_stride=256, q_out_stride=256, k_out_stride=256,
                            status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == RANGE
    got, live = host(buf).reshape(6, 4, 64), pos < 10
    assert np.array_equal(got[~live], x[~live])
    val, mag = ref.norm_rope(x[live], None, 0, cos[pos[live]], sin[pos[live]])
    assert np.all(np.abs(got[live] - val) <= row_bound(val, mag, "f32"))


def test_norm_rope_infinite_and_nan_rows_stay_apart(pkg, torch):
    x = np.ones((3, 2, 64), np.float32)
    x[1, 0, 5], x[1, 1, 7] = np.inf, np.nan
    g = np.ones(64, np.float32)
    buf, dg = dev(torch, x.reshape(3, -1)), dev(torch, g)
    out = torch.empty_like(buf)
    pkg.engine.qk_norm_rope(buf.data_ptr(), None, out.data_ptr(), None, 3, 2, 0, 64, None, None, None, 0, 0, dg.data_ptr())
    got = host(out).reshape(3, 2, 64)
    assert np.isfinite(got[[0, 2]]).all() and np.isnan(got[1, 1]).all()
    assert np.isnan(got[1, 0, 5]) and np.all(got[1, 0, :5] == 0)  # inf * 0 and 1 * 0, as the formula has it


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,page,layout,hq,hk,d,r,gains", [
    ([1], [1], 16, "head", 16, 4, 128, 64, False), ([1, 1, 1], [17, 16, 33], 16, "slot", 16, 4, 128, 64, True),
    ([5, 0, 1, 12], [5, 9, 40, 12], 7, "head", 0, 3, 64, 32, True), ([37, 21], [37, 150], 1, "slot", 6, 2, 64, 16, False),
    ([300, 211], [411, 211], 64, "slot", 16, 4, 128, 64, True), ([2] * 70, [3 + s for s in range(70)], 8, "head", 4, 1, 128, None, False)])
def test_append(pkg, torch, t, kv, new, total, page, layout, hq, hk, d, r, gains):
    rng = np.random.default_rng(len(new) * 7 + page)
    b = ref.Batch(rng, new, total, page, extra_rows=3)
    x = ref.round_to(rng.standard_normal((b.rows, hq + 2 * hk, d)) * 3, t)
    g = [rng.uniform(0.5, 2, d).astype(np.float32) if gains else None for _ in range(2)]
    top = max(total) + 1
    cos, sin = tables(rng, top, r or 8)
    before = [ref.round_to(rng.standard_normal((b.pages, page, hk, d)), kv) for _ in range(2)]
    pool, m = Pool(torch, kv, b, hk, d, layout, before, gap=8), Meta(torch, b)
    buf = dev(torch, x.reshape(b.rows, -1)).to(tt(torch, t))
    qo = torch.full((b.rows, hq * d), -7.0, dtype=buf.dtype, device="cuda")
    dc, ds = dev(torch, cos), dev(torch, sin)
    dg = [None if y is None else dev(torch, y) for y in g]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    e, wide, at = buf.element_size(), buf.shape[1], buf.data_ptr()
    ptr = lambda z: None if z is None else z.data_ptr()  # noqa: E731
    pkg.engine.paged_append(at + hq * d * e, at + (hq + hk) * d * e, b.rows, hk, d, **pool.args(), **m.kw,
                            q_ptr=at if hq else None, q_out_ptr=qo.data_ptr() if hq else None, q_heads=hq,
                            cos_ptr=ptr(dc) if r else None, sin_ptr=ptr(ds) if r else None, rope_rows=top,
                            rope_half_dim=r or 0, q_gamma_ptr=ptr(dg[0]), k_gamma_ptr=ptr(dg[1]), dtype=t,
                            q_stride=wide, k_stride=wide, v_stride=wide, status_ptr=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    kp, vp = pool.values()
    want_k, want_v = before[0].copy(), before[1].copy()
    bound_k = np.zeros_like(want_k)
    for s in range(b.seqs):
        for i in range(b.new[s]):
            p, row = b.total[s] - b.new[s] + i, b.start[s] + i
            pg, sl = b.place(s, p)
            val, mag = ref.norm_rope(x[row:row + 1, :hq + hk], None, 0, cos[p:p + 1] if r else None, sin[p:p + 1] if r else None)
            if gains:
                parts = [ref.norm_rope(x[row:row + 1, a:z], gm, 1e-6, cos[p:p + 1] if r else None, sin[p:p + 1] if r else None)
                         for a, z, gm in ((0, hq, g[0]), (hq, hq + hk, g[1]))]
                val, mag = (np.concatenate([u[j] for u in parts], 1) for j in (0, 1))
            want_k[pg, sl], bound_k[pg, sl] = val[0, hq:], row_bound(val, mag, kv)[0, hq:]
            want_v[pg, sl] = ref.round_to(x[row, hq + hk:], kv)
            if hq:
                assert np.all(np.abs(host(qo[row]).reshape(hq, d) - val[0, :hq]) <= row_bound(val, mag, t)[0, :hq])
    assert np.array_equal(vp, want_v)
    assert np.all(np.abs(kp - want_k) <= bound_k)  # everything else is as it was
    assert np.all(host(qo[b.rows - 3:]) == -7.0)  # rows of no sequence
    assert all(torch.isnan(z[..., d:]).all() for z in pool.t)


def test_append_skips_what_has_no_place(pkg, torch):
    """Bad page ids, lengths that do not fit, row ranges outside the rows, positions behind
    the tables: nothing is written for them, the status says so, the rest is right."""
    rng = np.random.default_rng(3)
    b = ref.Batch(rng, [1] * 8, [4, 4, 4, 4, 4, 4, 4, 4], 4, wide=2)
    b.table[:, 1] = b.free[0]
    b.table[1, 0], b.table[2, 0] = -1, b.pages  # no such pages
    b.len[3], b.len[4], b.len[5], b.len[6] = 9, 0, -3, 2**31 - 1  # two pages hold 8; no place for a row; none; none
    x = rng.standard_normal((8, 2, 64)).astype(np.float32)
    before = [rng.standard_normal((b.pages, 4, 1, 64)).astype(np.float32) for _ in range(2)]
    for bad in ("pages", "rows"):
        pool = Pool(torch, "f32", b, 1, 64, "slot", before)
        m, buf, st = Meta(torch, b), dev(torch, x.reshape(8, -1)), torch.zeros(1, dtype=torch.int32, device="cuda")
        want = [z.copy() for z in before]
        rows = 8
        if bad == "rows":
            m.start.copy_(dev(torch, np.array([-2, 1, 2, 9, 1, 0, 6, 7, 100], np.int32)))
        else:
            for s in (0, 7):
                pg, sl = b.place(s, 3)
                want[0][pg, sl, 0], want[1][pg, sl, 0] = x[s, 0], x[s, 1]
        pkg.engine.paged_append(buf.data_ptr(), buf.data_ptr() + 256, rows, 1, 64, **pool.args(), **m.kw, k_stride=128,
                                v_stride=128, status_ptr=st.data_ptr())
        torch.cuda.synchronize()
        assert int(st.item()) == RANGE
        if bad == "pages":
            assert all(np.array_equal(u, w) for u, w in zip(pool.values(), want))


def test_append_rounds_to_nearest_even_and_overflows_to_infinity(pkg, torch):
    b = ref.Batch(np.random.default_rng(0), [1], [1], 4)
    x = np.zeros((1, 2, 64), np.float32)
    x[0, 1, :6] = [65519.0, 65520.0, -1e30, 1 + 2.0**-11, 1 + 3 * 2.0**-11, np.nan]
    pool, m, buf = Pool(torch, "f16", b, 1, 64, "head"), Meta(torch, b), dev(torch, x.reshape(1, -1))
    pkg.engine.paged_append(buf.data_ptr(), buf.data_ptr() + 256, 1, 1, 64, **pool.args(), **m.kw, k_stride=128, v_stride=128)
    pg, sl = b.place(0, 0)
    v = pool.values()[1][pg, sl, 0]
    assert list(v[:5]) == [65504.0, np.inf, -np.inf, 1.0, 1 + 2.0**-9] and np.isnan(v[5])


# ---------------------------------------------------------------- attention
def attend(pkg, torch, b, q, pool, t, window=0, scale=None, max_q=None, stream=None, work=None, lse=True, pad=0, qpad=0, m=None):
    """q [rows][hq][d] float64 of type t's values; returns out, lse (float64), status."""
    rows, hq, d = q.shape
    m = m or Meta(torch, b)
    dq = torch.full((rows, hq * d + qpad), float("nan"), dtype=tt(torch, t), device="cuda")
    dq[:, :hq * d] = dev(torch, q.reshape(rows, -1)).to(dq.dtype)
    out = torch.full((rows, hq * d + pad), -7.0, dtype=dq.dtype, device="cuda")
    dl = torch.full((rows, hq), -7.0, dtype=torch.float32, device="cuda")
    if work is None:
        work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda").fill_(255)  # NaN as f32
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.engine.paged_attention(dq.data_ptr(), out.data_ptr(), rows, hq, pool.hk, d, **pool.args(), **m.kw,
                               max_q=max_q or max(1, max(b.new)), work_ptr=work.data_ptr(), scale=scale, window=window,
                               lse_ptr=dl.data_ptr() if lse else None, dtype=t, q_stride=hq * d + qpad,
                               out_stride=hq * d + pad, status_ptr=st.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    got = host(out)
    assert np.all(got[:, hq * d:] == -7.0)
    return got[:, :hq * d].reshape(rows, hq, d), host(dl), int(st.item())


def make(torch, rng, t, kv, new, total, page, layout, hq, hk, d, extra=2, qmul=1.5, gap=0, wide=None):
    b = ref.Batch(rng, new, total, page, extra_rows=extra, wide=wide)
    q = ref.round_to(rng.standard_normal((b.rows, hq, d)) * qmul, t)
    pages = [ref.round_to(rng.standard_normal((b.pages, page, hk, d)), kv) for _ in range(2)]
    used = np.zeros((b.pages, page), bool)
    for s in range(b.seqs):
        for p in range(b.total[s]):
            used[b.place(s, p)] = True
    for z in pages:  # stale slots hold anything
        z[~used] = np.nan
        if (~used).any():
            z[tuple(np.argwhere(~used)[0])] = np.inf
    return b, q, pages, Pool(torch, kv, b, hk, d, layout, pages, gap=gap)


def check_attention(b, got, gl, q, pages, t, kv, scale, window, bad=(), lse=True):
    out, wl, mass, size = ref.attention(b, q, *pages, scale, window, bad)
    owned = ~np.isnan(wl[:, 0])
    bound, lb = ref.attention_bounds(b, out, mass, size, t, kv, q.shape[2])
    err = np.abs(got - out)[owned]
    assert np.all(err <= bound[owned]), float(np.max(err / bound[owned]))
    assert np.all(got[~owned] == -7.0)
    if lse:
        empty = np.isneginf(wl) & owned[:, None]
        assert np.array_equal(np.isneginf(gl), empty)
        fin = owned[:, None] & ~empty
        assert np.all(np.abs(gl[fin] - wl[fin]) <= lb[fin] + 2.0**-23 * np.abs(wl[fin]))
        assert np.all(gl[~owned] == -7.0)


SHAPES = [
    # new, total, page, layout, hq, hk, d, window
    ([1], [1], 16, "head", 16, 4, 128, 0),
    ([1], [700], 16, "slot", 16, 4, 128, 0),
    ([1, 1, 1, 1, 1], [17, 16, 1, 129, 300], 16, "head", 16, 4, 128, 0),
    ([1] * 9, [3, 64, 65, 127, 128, 250, 5, 90, 31], 8, "slot", 4, 4, 64, 0),
    ([1, 1], [500, 131], 7, "head", 24, 3, 128, 100),
    ([1, 0, 1], [257, 50, 40], 1, "slot", 16, 1, 64, 0),
    ([4, 2, 3], [260, 2, 131], 32, "slot", 16, 4, 128, 0),
    ([3, 1], [64, 200], 20, "head", 2, 2, 128, 33),
    ([16, 5], [150, 5], 64, "head", 1, 1, 64, 0),
    ([40], [40], 16, "slot", 16, 4, 128, 0),
    ([70, 1, 33], [200, 140, 33], 16, "head", 8, 2, 128, 0),
    ([129], [300], 128, "slot", 4, 1, 64, 0),
    ([50, 65], [180, 190], 20, "slot", 6, 2, 128, 70),
    ([90], [260], 16, "head", 3, 3, 64, 7),
    ([5], [300], 16, "head", 128, 2, 64, 0),
    ([140], [3], 16, "slot", 4, 2, 64, 0),           # more new rows than positions: the first 137 attend to nothing
    ([3, 2], [1, 0], 16, "slot", 4, 2, 128, 0),      # the same for single tiles; a sequence without any position
]


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(pkg, torch, t, kv, shape):
    new, total, page, layout, hq, hk, d, window = shape
    rng = np.random.default_rng(sum(new) * 31 + sum(total))
    b, q, pages, pool = make(torch, rng, t, kv, new, total, page, layout, hq, hk, d, gap=8 if page == 20 else 0)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window, pad=16, qpad=8)
    assert st == 0
    check_attention(b, got, gl, q, pages, t, kv, d ** -0.5, window)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total", [([1], [900]), ([60], [170])])
def test_attention_peaked_and_flat_scores(pkg, torch, t, kv, new, total):
    """A large scale (one position takes all, late maxima) and a tiny one (all alike)."""
    rng = np.random.default_rng(8)
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "head", 4, 1, 128)
    for scale in (3.0, 1e-6):
        got, gl, st = attend(pkg, torch, b, q, pool, t, scale=scale)
        check_attention(b, got, gl, q, pages, t, kv, float(np.float32(scale)), 0)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total", [([1, 1], [400, 90]), ([4], [130]), ([70], [150])])
def test_attention_masks_bad_pages(pkg, torch, t, kv, new, total):
    rng = np.random.default_rng(9)
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "slot", 8, 2, 128)
    for bad in (-1, b.pages, 2**31 - 1, -2**31):
        b.table[0, 1] = b.table[0, 4] = bad
        got, gl, st = attend(pkg, torch, b, q, pool, t)
        assert st == RANGE
        check_attention(b, got, gl, q, pages, t, kv, 128 ** -0.5, 0, bad=(bad,))
    b.table[:] = -5  # nothing but bad pages: every row attends to nothing
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    owned = int(b.start[-1])
    assert st == RANGE and np.all(got[:owned] == 0) and np.all(np.isneginf(gl[:owned]))


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 50])
def test_attention_skips_what_is_out_of_range(pkg, torch, t, kv, n):
    """Lengths that do not fit the table, row ranges outside the rows, more new rows than
    max_q: their rows stay as they were; the sequences beside them are right."""
    rng = np.random.default_rng(10)
    b, q, pages, pool = make(torch, rng, t, kv, [n] * 4, [100, 80, 60, 100], 16, "slot", 4, 2, 64, wide=8)
    for lens in ([100, 129, 60, 100], [100, -1, 60, 100], [100, 2**31 - 1, 60, 100]):
        b2 = ref.Batch(np.random.default_rng(0), b.new, b.total, 16)
        b2.start, b2.table, b2.rows, b2.pages, b2.wide = b.start, b.table, b.rows, b.pages, b.wide
        b2.len = np.array(lens, np.int32)
        got, gl, st = attend(pkg, torch, b2, q, pool, t)
        assert st == RANGE
        assert np.all(got[n:2 * n] == -7.0) and np.all(gl[n:2 * n] == -7.0)
        got[n:2 * n] = gl[n:2 * n] = 0
        b3 = ref.Batch(np.random.default_rng(0), b.new, b.total, 16)
        b3.start, b3.table, b3.rows = b.start, b.table, b.rows
        out, wl, mass, size = ref.attention(b3, q, *pages, 64 ** -0.5, 0)
        bound, _ = ref.attention_bounds(b3, out, mass, size, t, kv, 64)
        keep = [r for r in range(4 * n) if not n <= r < 2 * n]
        assert np.all(np.abs(got - out)[keep] <= bound[keep])
    m = Meta(torch, b)
    m.start.copy_(dev(torch, np.array([-1, n, 2 * n, 3 * n, 2**31 - 1], np.int32)))  # the first and the last range
    got, gl, st = attend(pkg, torch, b, q, pool, t, m=m)
    assert st == RANGE and np.all(got[:n] == -7.0) and np.all(got[3 * n:] == -7.0) and np.all(got[n:3 * n] != -7.0)
    if n > 1:
        b.new = [n] * 4
        got, gl, st = attend(pkg, torch, b, q, pool, t, max_q=n - 1)
        assert st == RANGE and np.all(got == -7.0)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,hq", [([3], [70], 4), ([64], [200], 4), ([100], [100], 2)])
def test_attention_infinite_values_reach_only_rows_that_see_them(pkg, torch, t, kv, new, total, hq):
    """K and V of a new position hold infinities and NaN: rows before it do not notice; rows
    from it on get what the formula gives (weights are positive: the infinity, or NaN)."""
    rng = np.random.default_rng(11)
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "head", hq, 1, 64, qmul=0.5)
    n, L = new[0], total[0]
    pv = L - n + n // 2
    pg, sl = b.place(0, pv)
    pages[1][pg, sl, 0, 5], pages[1][pg, sl, 0, 9] = np.inf, np.nan
    pool = Pool(torch, kv, b, 1, 64, "head", pages)
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    clean = [pages[0], pages[1].copy()]
    clean[1][pg, sl, 0, [5, 9]] = 0
    rest = [x for x in range(64) if x not in (5, 9)]
    out, wl, mass, size = ref.attention(b, q, *clean, 64 ** -0.5, 0)
    bound, _ = ref.attention_bounds(b, out, mass, size, t, kv, 64)
    before, after = slice(0, n // 2), slice(n // 2, n)
    assert np.all(np.abs(got - out)[before] <= bound[before])
    assert np.all(np.abs(got - out)[after][..., rest] <= bound[after][..., rest])
    assert np.all(np.isposinf(got[after][..., 5])) and np.all(np.isnan(got[after][..., 9]))
    # K: the rows that see the NaN are NaN, the others are not
    pages[1][pg, sl, 0, [5, 9]] = 0
    pages[0][pg, sl, 0, 3] = np.nan
    got, gl, st = attend(pkg, torch, b, q, Pool(torch, kv, b, 1, 64, "head", pages), t)
    assert np.all(np.abs(got - out)[before] <= bound[before])
    assert np.all(np.isnan(got[after])) and np.all(np.isnan(gl[after])) and np.isfinite(gl[before]).all()
    # q: a NaN row is NaN, its neighbours are not
    pages[0][pg, sl, 0, 3] = 0
    q2 = q.copy()
    q2[1, 0, 7] = np.nan
    got, gl, st = attend(pkg, torch, b, q2, Pool(torch, kv, b, 1, 64, "head", pages), t)
    assert np.all(np.isnan(got[1, 0])) and np.isfinite(got[0]).all() and np.isfinite(got[2:n]).all() and np.isfinite(got[1, 1:]).all()


def check_on_gpu(torch, b, got, gl, q, pool, t, kv, window=0):
    """check_attention in 64 bits on the GPU, for more positions than numpy loops take."""
    hq, d, hk = q.shape[1], q.shape[2], pool.hk
    for s in range(b.seqs):
        L, n = b.total[s], b.new[s]
        pg = torch.from_numpy(b.table[s, :-(-L // b.page)].astype(np.int64)).cuda()
        k, v = (z.double()[pg][..., :d] for z in pool.t)
        k, v = ((z if pool.layout == "slot" else z.transpose(1, 2)).reshape(-1, hk, d)[:L] for z in (k, v))
        p, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        hide = (j > p) | (j <= p - window) if window else j > p
        for h in range(hq):
            rows, g = slice(b.start[s], b.start[s] + n), h // (hq // hk)
            x = torch.from_numpy(q[rows, h]).cuda() @ k[:, g].T * d ** -0.5
            x[hide] = -np.inf
            w = torch.softmax(x, 1)
            out, mass = (w @ v[:, g]).cpu().numpy(), (w @ v[:, g].abs()).cpu().numpy()
            size = (torch.from_numpy(np.abs(q[rows, h])).cuda() @ k[:, g].abs().T * d ** -0.5).masked_fill(hide, 0).amax(1).cpu().numpy()
            bound, lb = ref.attention_bounds(b, out, mass, size, t, kv, d)
            err = np.abs(got[rows, h] - out)
            assert np.all(err <= bound), (s, h, float(np.max(err / bound)))
            wl = torch.logsumexp(x, 1).cpu().numpy()
            assert np.all(np.abs(gl[rows, h] - wl) <= lb + 2.0**-23 * np.abs(wl))


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,total,page,layout,hq,hk,d,window", [
    ([1, 1], [9001, 300], 16, "slot", 8, 2, 128, 0),               # split over the positions
    ([40, 40], [9001, 300], 16, "slot", 8, 2, 128, 0),
    ([70] * 20, [1500 - 61 * s for s in range(20)], 64, "head", 16, 4, 128, 0),  # many tiles in one piece
    ([33, 1, 200, 7] * 10, [700, 1300, 410, 900] * 10, 32, "slot", 8, 4, 64, 0),
    ([90] * 16, [1200] * 16, 128, "slot", 16, 4, 64, 500),         # pages longer than a tile
    ([90] * 16, [900] * 16, 24, "head", 12, 4, 128, 333),          # pages that no tile is made of
    ([600], [600], 256, "head", 6, 2, 128, 0),
    ([2] * 40, [31 * s + 2 for s in range(40)], 16, "head", 8, 2, 128, 0),
])
def test_attention_longer_caches(pkg, torch, t, kv, new, total, page, layout, hq, hk, d, window):
    """Work split over the positions, and pieces of many tiles, against 64 bits on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(len(new))
    b = ref.Batch(np.random.default_rng(1), new, total, page)
    pool = Pool(torch, kv, b, hk, d, layout)
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    q = ref.round_to(np.random.default_rng(2).standard_normal((b.rows, hq, d)) * 1.5, t)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    check_on_gpu(torch, b, got, gl, q, pool, t, kv, window)


@pytest.mark.parametrize("n,seqs", [(1, 2), (40, 1), (70, 20)])
@pytest.mark.parametrize("qs,ks,vs", [(1e-15, 1e15, 1.0), (1e12, 1e-12, 1e-30), (1.0, 1.0, 1e30), (1.0, 1.0, "steps"),
                                      (1.0, 1.0, "late"), (1.0, "steps", 1.0), (1.0, 1.0, "zeros"), (1.0, 1.0, "far"),
                                      (1.0, 1.0, "grows")])
def test_attention_f32_cache_of_any_size(pkg, torch, n, seqs, qs, ks, vs):
    """f32 caches whose values lie far from 1, or whose tiles differ in size: "steps": every 64
    positions another magnitude, "late": large values at the end alone, "zeros": tiles of zeros,
    "far": late values that are 1e45 times as large, "grows": 1000 times as large every 64."""
    g = torch.Generator(device="cuda").manual_seed(n)
    total = [900 + s for s in range(seqs)]
    b = ref.Batch(np.random.default_rng(1), [n] * seqs, total, 16)
    pool = Pool(torch, "f32", b, 4, 128, "slot")
    size = {"steps": lambda p: 10.0 ** (3.0 * ((p // 64) % 5) - 8), "late": lambda p: np.where(p < 850, 1.0, 1e9),
            "zeros": lambda p: np.where((p // 64) % 3 == 0, 0.0, 1.0),
            "far": lambda p: np.where(p < 832 + 64 * (p[-1] > 910), 1e-20, 1e25), "grows": lambda p: 10.0 ** (3.0 * (p // 64) - 20)}
    for z, f in zip(pool.t, (ks, vs)):
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
        for s in range(seqs):
            p = np.arange(total[s])
            f_p = size[f](p) if isinstance(f, str) else np.full(total[s], f)
            pg = torch.from_numpy(b.table[s, p // 16].astype(np.int64)).cuda()
            z[pg, torch.from_numpy(p % 16).cuda()] *= torch.from_numpy(f_p).float().cuda()[:, None, None]
    q = ref.round_to(np.random.default_rng(2).standard_normal((b.rows, 16, 128)) * qs * (1e-3 if ks == "steps" else 1.0), "f32")
    got, gl, st = attend(pkg, torch, b, q, pool, "f32")
    assert st == 0
    check_on_gpu(torch, b, got, gl, q, pool, "f32", "f32")


@pytest.mark.parametrize("qs", [1e-30, 1e-6, 1e6, 3e30])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_f32_rows_of_any_size(pkg, torch, n, qs):
    rng = np.random.default_rng(4)
    b, q, pages, pool = make(torch, rng, "f32", "f16", [n], [200], 16, "slot", 4, 1, 64, extra=0)
    q = ref.round_to(q * qs, "f32")
    scale = float(np.float32(0.125 / qs)) if qs != 1e-30 else 0.125
    got, gl, st = attend(pkg, torch, b, q, pool, "f32", scale=scale)
    check_attention(b, got, gl, q, pages, "f32", "f16", scale, 0)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 30])
def test_attention_of_sequences_that_share_pages(pkg, torch, t, kv, n):
    rng = np.random.default_rng(6)
    b, q, pages, pool = make(torch, rng, t, kv, [n] * 3, [100, 90, 64], 16, "head", 4, 2, 64)
    b.table[1, :4], b.table[2, :4] = b.table[0, :4], b.table[0, :4]
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    assert st == 0
    check_attention(b, got, gl, q, pages, t, kv, 0.125, 0)


@pytest.mark.parametrize("t,kv", TYPES)
def test_attention_overlapping_row_ranges_stay_in_bounds(pkg, torch, t, kv):
    """Row ranges that fall back: more tiles than the rows can have. Nothing is written."""
    rng = np.random.default_rng(7)
    b, q, pages, pool = make(torch, rng, t, kv, [320, 320], [320, 320], 16, "slot", 2, 1, 64, extra=0)
    b.start = np.array([0, 640, 0, 640, 0, 640, 0, 640, 0], np.int32)
    b.seqs, b.len = 8, np.full(8, 640, np.int32)
    b.table = np.tile(np.arange(40, dtype=np.int32), (8, 1))
    b.wide, b.new = 40, [640] * 8
    got, gl, st = attend(pkg, torch, b, q, pool, t)
    assert st == RANGE and np.all(got == -7.0) and np.all(gl == -7.0)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("new,window", [([1] * 40 + [300, 150], 0), ([1, 2, 0, 70, 1, 3, 500, 2] * 5, 200), ([2, 400], 0),
                                        ([5, 1, 4, 3, 2] * 9, 0), ([700] + [0] * 60 + [1], 0)])
def test_attention_single_tokens_and_chunks_together(pkg, torch, t, kv, new, window):
    """One call with single tokens, short runs and long chunks, in any order."""
    rng = np.random.default_rng(len(new))
    total = [n + int(rng.integers(0, 1200)) for n in new]
    b = ref.Batch(rng, new, total, 16)
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = Pool(torch, kv, b, 4, 64, "slot")
    for z in pool.t:
        z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    q = ref.round_to(rng.standard_normal((b.rows, 8, 64)) * 1.5, t)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    check_on_gpu(torch, b, got, gl, q, pool, t, kv, window)


def test_attention_page_offsets_past_32_bits(pkg, torch):
    """A pool of more than 2^32 bytes (and elements past 2^31): pages at its far end."""
    page, hk, d, pages = 64, 4, 128, 70000
    pool_t = [torch.empty((pages, page, hk, d), dtype=torch.float16, device="cuda") for _ in range(2)]
    b = ref.Batch(np.random.default_rng(3), [1, 30], [100, 90], page)
    far = np.array([pages - 1, pages - 7, 3, 66000], np.int32)
    b.table = far.reshape(2, 2).copy()
    b.pages, b.wide = pages, 2
    rng = np.random.default_rng(4)
    small = [ref.round_to(rng.standard_normal((4, page, hk, d)), "f16") for _ in range(2)]
    for z, f in zip(pool_t, small):
        z[torch.from_numpy(far.astype(np.int64)).cuda()] = dev(torch, f).half()
    pool = Pool.__new__(Pool)
    pool.t, pool.b, pool.hk, pool.d, pool.kv, pool.strides = pool_t, b, hk, d, "f16", (page * hk * d, d, hk * d)
    q = ref.round_to(rng.standard_normal((b.rows, 8, d)), "f32")
    got, gl, st = attend(pkg, torch, b, q, pool, "f32")
    b2 = ref.Batch(np.random.default_rng(3), b.new, b.total, page)
    b2.table = np.array([[0, 1], [2, 3]], np.int32)
    check_attention(b2, got, gl, q, small, "f32", "f16", d ** -0.5, 0)
    k = torch.ones((b.rows, hk * d), device="cuda")
    m = Meta(torch, b)
    pkg.engine.paged_append(k.data_ptr(), k.data_ptr(), b.rows, hk, d, **pool.args(), **m.kw)
    torch.cuda.synchronize()
    assert all(bool((z[pages - 7, 35] == 1).all()) and bool((z[pages - 7, 36] != 1).any()) for z in pool_t)


@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("n", [1, 3, 80])
def test_attention_is_deterministic_and_needs_no_lse(pkg, torch, t, kv, n):
    rng = np.random.default_rng(12)
    b, q, pages, pool = make(torch, rng, t, kv, [n, n], [3000, 500], 16, "slot", 8, 2, 128)
    a = attend(pkg, torch, b, q, pool, t)
    work = torch.zeros(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    c = attend(pkg, torch, b, q, pool, t, work=work, lse=False)
    e = attend(pkg, torch, b, q, pool, t, work=work)
    assert np.array_equal(a[0], c[0]) and np.array_equal(a[0], e[0]) and np.array_equal(a[1], e[1]) and np.all(c[1] == -7.0)


# ---------------------------------------------------------------- together, as a server runs them
@pytest.mark.parametrize("t,kv", TYPES)
def test_prompt_then_tokens_captured(pkg, torch, t, kv):
    """Prompts of three requests in one pass, then single tokens as a replayed CUDA graph
    whose lengths grow on the device, on a stream of their own: append with norms and
    rotation, then attention, against the 64-bit forms on the values that lie in the pages."""
    rng = np.random.default_rng(13)
    hq, hk, d, page, steps = 8, 2, 128, 16, 5
    prompt = [37, 5, 64]
    final = [x + steps for x in prompt]
    b = ref.Batch(rng, prompt, prompt, page, wide=6)
    full = ref.Batch(np.random.default_rng(1), prompt, final, page, wide=6)
    cos, sin = tables(rng, 128, 64)
    g = [rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2)]
    dc, ds, dg = dev(torch, cos), dev(torch, sin), [dev(torch, y) for y in g]
    pool = Pool(torch, kv, full, hk, d, "head")
    work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    w = (hq + 2 * hk) * d

    def step(x, qr, out, m, rows, max_q, stream):
        e, at = x.element_size(), x.data_ptr()
        pkg.engine.paged_append(at + hq * d * e, at + (hq + hk) * d * e, rows, hk, d, **pool.args(), **m.kw, q_ptr=at,
                                q_out_ptr=qr.data_ptr(), q_heads=hq, cos_ptr=dc.data_ptr(), sin_ptr=ds.data_ptr(),
                                rope_rows=128, rope_half_dim=64, q_gamma_ptr=dg[0].data_ptr(), k_gamma_ptr=dg[1].data_ptr(),
                                dtype=t, q_stride=w, k_stride=w, v_stride=w, stream=stream)
        pkg.engine.paged_attention(qr.data_ptr(), out.data_ptr(), rows, hq, hk, d, **pool.args(), **m.kw, max_q=max_q,
                                   work_ptr=work.data_ptr(), dtype=t, stream=stream)

    def check(b, x, out):
        kp, vp = pool.values()
        xs = host(x).reshape(b.rows, hq + 2 * hk, d)
        pos = np.concatenate([np.arange(L - n, L) for n, L in zip(b.new, b.total)])
        q, _ = ref.norm_rope(xs[:, :hq], g[0], 1e-6, cos[pos], sin[pos])
        k, mag = ref.norm_rope(xs[:, hq:hq + hk], g[1], 1e-6, cos[pos], sin[pos])
        row = 0
        for s in range(b.seqs):
            for i in range(b.new[s]):
                pg, sl = b.place(s, b.total[s] - b.new[s] + i)
                assert np.all(np.abs(kp[pg, sl] - k[row]) <= row_bound(k, mag, kv)[row])
                assert np.array_equal(vp[pg, sl], ref.round_to(xs[row, hq + hk:], kv))
                row += 1
        q = ref.round_to(q, t)  # may be a step off what the kernel wrote: one more step on q in the bound
        want, _, mass, size = ref.attention(b, q, kp, vp, d ** -0.5, 0)
        bound, _ = ref.attention_bounds(b, want, mass, size, t, kv, d)
        bound += 2 * (2 * ref.HALF_STEP[t] * size)[..., None] * mass
        assert np.all(np.abs(host(out).reshape(want.shape) - want) <= bound)

    b.table = full.table
    m = Meta(torch, b)
    x = torch.randn(b.rows, w, device="cuda").to(tt(torch, t))
    qr, out = (torch.empty(b.rows, hq * d, dtype=x.dtype, device="cuda") for _ in range(2))
    side.wait_stream(torch.cuda.current_stream())
    step(x, qr, out, m, b.rows, max(prompt), side)
    torch.cuda.synchronize()
    check(b, x, out)

    one = ref.Batch(np.random.default_rng(2), [1, 1, 1], final, page, wide=6)
    one.table = full.table
    m1 = Meta(torch, one)
    m1.len.copy_(m.len)
    x1 = torch.zeros(3, w, dtype=x.dtype, device="cuda")
    q1, o1 = (torch.empty(3, hq * d, dtype=x.dtype, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m1.len += 1
        step(x1, q1, o1, m1, 3, 1, torch.cuda.current_stream())
    for i in range(steps):
        x1.copy_(torch.randn(3, w, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        one.total = [p + i + 1 for p in prompt]
        check(one, x1, o1)


def test_two_streams_with_a_workspace_each(pkg, torch):
    """Two captured calls replayed at the same time on two streams give what each gives alone."""
    rng = np.random.default_rng(14)
    runs = []
    for n, total in ((1, 5000), (60, 3000)):
        b, q, pages, pool = make(torch, rng, "f32", "f16", [n], [total], 16, "slot", 8, 2, 128, extra=0)
        m, dq = Meta(torch, b), dev(torch, q.reshape(b.rows, -1)).float()
        out = torch.zeros_like(dq)
        work = torch.empty(pkg.engine.PAGED_WORK_BYTES, dtype=torch.uint8, device="cuda")
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            pkg.engine.paged_attention(dq.data_ptr(), out.data_ptr(), b.rows, 8, 2, 128, **pool.args(), **m.kw, max_q=n,
                                       work_ptr=work.data_ptr(), stream=side)
        graph.replay()
        torch.cuda.synchronize()
        runs.append((graph, side, out, out.clone(), (pool, m, dq, work)))
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, side, _, _, _ in runs:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone) for _, _, out, alone, _ in runs)
