"""The paged-cache entry points without a GPU: what the host refuses, before any launch,
and the plain 64-bit forms that the GPU tests compare with."""
import numpy as np
import pytest

import paged_ref as ref

INVALID, UNSUPPORTED = 1, 7
A = 1 << 20  # an aligned address that no refused call reads


@pytest.fixture(scope="module", autouse=True)
def built(pkg):
    import importlib
    importlib.import_module("qora-llm_b200.build").build()


def norm_args(**kw):
    a = dict(q_ptr=A, k_ptr=A, q_out_ptr=A, k_out_ptr=A, rows=3, q_heads=8, kv_heads=2, head_dim=128, pos_ptr=A,
             cos_ptr=A, sin_ptr=A, rope_rows=64, rope_half_dim=64)
    a.update(kw)
    return a


def append_args(**kw):
    a = dict(k_ptr=A, v_ptr=A, rows=3, kv_heads=2, head_dim=128, k_pages_ptr=A, v_pages_ptr=A, num_pages=10,
             page_size=16, q_start_ptr=A, kv_len_ptr=A, table_ptr=A, table_stride=4, seqs=2)
    a.update(kw)
    return a


def attend_args(**kw):
    a = dict(q_ptr=A, out_ptr=A, rows=3, q_heads=8, kv_heads=2, head_dim=128, k_pages_ptr=A, v_pages_ptr=A,
             num_pages=10, page_size=16, q_start_ptr=A, kv_len_ptr=A, table_ptr=A, table_stride=4, seqs=2, max_q=2,
             work_ptr=A)
    a.update(kw)
    return a


PAGES = [
    (dict(k_pages_ptr=None), INVALID, "NULL"), (dict(v_pages_ptr=A + 8), INVALID, "16 bytes"),
    (dict(num_pages=0), INVALID, "0 pages"), (dict(page_size=0), INVALID, "pages of 0"),
    (dict(page_strides=(4096, 2048, 64)), INVALID, "overlap"), (dict(page_strides=(2048, 2048, 128)), INVALID, "overlap"),
    (dict(page_strides=(4096, 2048, 129)), INVALID, "16 bytes"), (dict(page_strides=(4096, 100, 128)), INVALID, "overlap"),
    (dict(page_strides=(1 << 50, 2048, 128)), INVALID, "2\\^40"),
    (dict(q_start_ptr=None), INVALID, "batch"), (dict(kv_len_ptr=None), INVALID, "batch"),
    (dict(table_ptr=None), INVALID, "batch"), (dict(table_stride=0), INVALID, "table rows"),
    (dict(table_stride=1 << 30), INVALID, "table rows"), (dict(seqs=1 << 21), INVALID, "sequences"),
    (dict(kv_dtype="bf16"), UNSUPPORTED, "cache of type"), (dict(dtype="f16"), UNSUPPORTED, "cache of type"),
    (dict(head_dim=96), UNSUPPORTED, "head_dim 96"), (dict(head_dim=0), UNSUPPORTED, "head_dim 0"),
    (dict(rows=-1), INVALID, "rows"), (dict(kv_heads=0), INVALID, "kv heads"),
]


def refused(pkg, fn, args, status, match):
    with pytest.raises(pkg.QoraError, match=match) as e:
        fn(**args)
    assert e.value.status == status


@pytest.mark.parametrize("kw,status,match", [
    (dict(q_ptr=None), INVALID, "q is NULL"), (dict(k_out_ptr=None), INVALID, "k_out is NULL"),
    (dict(q_ptr=A + 4), INVALID, "16-byte"), (dict(q_stride=1026), INVALID, "16-byte"),
    (dict(q_stride=512), INVALID, "row stride"), (dict(k_stride=64), INVALID, "row stride"),
    (dict(q_stride=2048, q_out_ptr=A), INVALID, "in place"), (dict(head_dim=80), UNSUPPORTED, "head_dim"),
    (dict(q_heads=0, kv_heads=0), INVALID, "no heads"), (dict(q_heads=2000), INVALID, "heads"),
    (dict(sin_ptr=None), INVALID, "go together"), (dict(pos_ptr=None), INVALID, "positions"),
    (dict(rope_half_dim=0), INVALID, "rope_half_dim"), (dict(rope_half_dim=72), INVALID, "rope_half_dim"),
    (dict(rope_half_dim=12), UNSUPPORTED, "multiple of 8"), (dict(rope_rows=0), INVALID, "rope_rows"),
    (dict(q_gamma_ptr=A, eps=float("nan")), INVALID, "eps"), (dict(q_gamma_ptr=A, eps=-1.0), INVALID, "eps"),
    (dict(k_gamma_ptr=A + 4), INVALID, "aligned"), (dict(cos_ptr=A + 4), INVALID, "aligned"),
    (dict(rows=1 << 25), INVALID, "rows"),
])
def test_norm_rope_refusals(pkg, kw, status, match):
    refused(pkg, pkg.engine.qk_norm_rope, norm_args(**kw), status, match)


@pytest.mark.parametrize("kw,status,match", PAGES + [
    (dict(k_ptr=None), INVALID, "k is NULL"), (dict(v_ptr=A + 2), INVALID, "16-byte"),
    (dict(v_stride=8), INVALID, "row stride"), (dict(q_heads=4), INVALID, "q is NULL"),
    (dict(q_heads=4, q_ptr=A), INVALID, "q_out is NULL"), (dict(cos_ptr=A), INVALID, "go together"),
    (dict(cos_ptr=A, sin_ptr=A, rope_half_dim=65, rope_rows=9), INVALID, "rope_half_dim"),
])
def test_append_refusals(pkg, kw, status, match):
    refused(pkg, pkg.engine.paged_append, append_args(**kw), status, match)


@pytest.mark.parametrize("kw,status,match", PAGES + [
    (dict(q_ptr=None), INVALID, "q is NULL"), (dict(out_ptr=None), INVALID, "out is NULL"),
    (dict(out_stride=1000), INVALID, "row stride"), (dict(q_heads=7), INVALID, "over"), (dict(q_heads=0), INVALID, "over"),
    (dict(q_heads=258), INVALID, "over"), (dict(scale=0.0), INVALID, "scale"), (dict(scale=-1.0), INVALID, "scale"),
    (dict(scale=float("nan")), INVALID, "scale"), (dict(scale=float("inf")), INVALID, "scale"),
    (dict(window=1 << 31), INVALID, "window"), (dict(max_q=0), INVALID, "max_q"), (dict(work_ptr=None), INVALID, "workspace"),
    (dict(work_ptr=A + 16), INVALID, "workspace"), (dict(work_bytes=1 << 20), INVALID, "workspace"),
])
def test_attention_refusals(pkg, kw, status, match):
    refused(pkg, pkg.engine.paged_attention, attend_args(**kw), status, match)


def test_nothing_to_do_launches_nothing(pkg):
    """No rows or no sequences: accepted without a device."""
    pkg.engine.qk_norm_rope(**norm_args(rows=0))
    pkg.engine.paged_append(**append_args(rows=0))
    pkg.engine.paged_append(**append_args(seqs=0))
    pkg.engine.paged_attention(**attend_args(rows=0))
    pkg.engine.paged_attention(**attend_args(seqs=0, max_q=0))


def test_empty_arrays_may_be_null(pkg):
    """Arrays without elements have no address: empty tensors give 0."""
    pkg.engine.qk_norm_rope(**norm_args(rows=0, q_ptr=None, k_ptr=None, q_out_ptr=None, k_out_ptr=None, pos_ptr=None))
    pkg.engine.paged_append(**append_args(rows=0, k_ptr=None, v_ptr=None))
    pkg.engine.paged_append(**append_args(rows=0, seqs=0, k_ptr=None, v_ptr=None, kv_len_ptr=None, table_ptr=None))
    pkg.engine.paged_attention(**attend_args(rows=0, q_ptr=None, out_ptr=None))
    pkg.engine.paged_attention(**attend_args(rows=0, seqs=0, max_q=0, q_ptr=None, out_ptr=None, kv_len_ptr=None, table_ptr=None))


M = 1 << 16  # bytes beyond the rows of the calls above


@pytest.mark.parametrize("fn,args,match", [
    ("qk_norm_rope", norm_args(q_out_ptr=A + 64, k_ptr=A + M, k_out_ptr=A + M), "q and its output"),
    ("qk_norm_rope", norm_args(k_ptr=A + M, k_out_ptr=A + M + 512), "k and its output"),
    ("qk_norm_rope", norm_args(k_ptr=A + 1024, k_out_ptr=A + M), "q_out and k overlap"),
    ("qk_norm_rope", norm_args(k_ptr=A + M, k_out_ptr=A + 4096, q_ptr=A, q_out_ptr=A + 2 * M), "k_out and q"),
    ("qk_norm_rope", norm_args(k_ptr=A + M, k_out_ptr=A + 2 * M, q_out_ptr=A + 2 * M), "q_out and k_out"),
    ("paged_append", append_args(q_heads=8, q_ptr=A + M, q_out_ptr=A + M + 16), "q and its output"),
    ("paged_append", append_args(q_heads=8, q_ptr=A + M, q_out_ptr=A, v_ptr=A + 2 * M), "q_out and k"),
    ("paged_append", append_args(q_heads=8, q_ptr=A + M, q_out_ptr=A, k_ptr=A + 2 * M), "q_out and v"),
    ("paged_attention", attend_args(), "q and out"), ("paged_attention", attend_args(out_ptr=A + 2 * 4096), "q and out"),
])
def test_overlapping_rows_are_refused(pkg, fn, args, match):
    refused(pkg, getattr(pkg.engine, fn), args, INVALID, match)


def test_parts_of_one_joined_row_do_not_overlap(pkg):
    """Accepted as far as the rows go: what refuses these calls is the last check."""
    w = (8 + 2 + 2) * 128
    joined = dict(q_stride=w, k_stride=w, dtype="f32")
    with pytest.raises(pkg.QoraError, match="go together"):
        pkg.engine.qk_norm_rope(**norm_args(**joined, k_ptr=A + 4096, k_out_ptr=A + 4096, q_out_stride=w, k_out_stride=w, sin_ptr=None))
    with pytest.raises(pkg.QoraError, match="pages of 0"):
        pkg.engine.paged_append(**append_args(**joined, q_heads=8, q_ptr=A, q_out_ptr=A, q_out_stride=w, k_ptr=A + 4096,
                                              v_ptr=A + 4096 + 1024, v_stride=w, page_size=0))
    with pytest.raises(pkg.QoraError, match="scale"):
        pkg.engine.paged_attention(**attend_args(q_stride=2048, out_ptr=A + 4096, out_stride=2048, scale=0.0))


@pytest.mark.parametrize("fn,args,match", [
    ("qk_norm_rope", norm_args(k_ptr=A + M, k_out_ptr=A + M, pos_ptr=A + 2), "4-byte"),
    ("paged_append", append_args(kv_len_ptr=A + 1), "4-byte"), ("paged_append", append_args(status_ptr=A + 2), "4-byte"),
    ("paged_attention", attend_args(out_ptr=A + M, lse_ptr=A + 2), "4-byte"),
    ("paged_attention", attend_args(out_ptr=A + M, table_ptr=A + 3), "4-byte"),
])
def test_misaligned_words_are_refused(pkg, fn, args, match):
    refused(pkg, getattr(pkg.engine, fn), args, INVALID, match)


def test_scale_that_leaves_f32(pkg):
    refused(pkg, pkg.engine.paged_attention, attend_args(scale=3e38), INVALID, "scale")


def test_unknown_element_type(pkg):
    with pytest.raises(ValueError, match="f8"):
        pkg.engine.paged_append(**append_args(dtype="f8"))


# ---------------------------------------------------------------- the plain forms themselves
def test_reference_norm_rope_turns_by_the_angle():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 16))
    ang = rng.uniform(0, 6, (3, 4))
    y, _ = ref.norm_rope(x, None, 0.0, np.cos(ang), np.sin(ang))
    z = (x[..., :4] + 1j * x[..., 4:8]) * np.exp(1j * ang)[:, None]
    assert np.allclose(y[..., :4], z.real) and np.allclose(y[..., 4:8], z.imag) and np.array_equal(y[..., 8:], x[..., 8:])
    g = rng.standard_normal(16)
    y, _ = ref.norm_rope(x, g, 0.0, None, None)
    assert np.allclose((y / g * (y / g)).mean(-1), 1.0)


def test_reference_attention_is_a_softmax_over_the_table():
    rng = np.random.default_rng(1)
    b = ref.Batch(rng, [2, 0, 1], [5, 3, 1], 2)
    kp, vp = (rng.standard_normal((b.pages, 2, 1, 8)) for _ in range(2))
    q = rng.standard_normal((b.rows, 2, 8))
    out, lse, _, _ = ref.attention(b, q, kp, vp, 0.5, 0)
    k = np.stack([kp[b.place(0, p)][0] for p in range(5)])
    v = np.stack([vp[b.place(0, p)][0] for p in range(5)])
    x = 0.5 * q[0, 1] @ k[:4].T  # the first new row of sequence 0 sits at position 3
    assert np.allclose(out[0, 1], np.exp(x) @ v[:4] / np.exp(x).sum()) and np.allclose(lse[0, 1], np.log(np.exp(x).sum()))
    assert np.allclose(out[2, 0], vp[b.place(2, 0)][0])


def test_rounding_helper():
    x = np.float32([1.0, 1 + 2.0**-9, 1 + 2.0**-8, -3.1415927, 65519.0, 65520.0])
    b = ref.round_to(x[:4], "bf16")
    assert np.all(np.abs(b - x[:4]) <= ref.HALF_STEP["bf16"] * np.abs(x[:4]))
    assert ref.round_to(x[4:], "f16")[0] == 65504.0 and np.isinf(ref.round_to(x[4:], "f16")[1])
