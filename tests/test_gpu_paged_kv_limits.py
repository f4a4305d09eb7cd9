"""Paged key/value cache on the GPU where its numbers reach their limits:
dominant scores, values that are not finite."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged_kv import T, U, Cache, _check_attend, _half_step, _kv, _normal, _reference, _run

pytestmark = pytest.mark.gpu


def _sink(c, gap, values):
    """Sequence 0 of `c` takes the given values and zero keys, but for one row: its key gives a query of
    (1, 0, ..) the score `gap`, and its value is zero."""
    n = c.lens[0]
    at = n // 3
    k, v = torch.zeros(c.kv_heads, n, c.dim), values
    k[:, at, 0] = gap
    v[:, at] = 0.0
    c.rows[0] = [k.to(T[c.dtype]), v.to(T[c.dtype])]
    c.put(0)


# head dims and groups of every tensor-core form: 8 and 16 rows, dims that fill a form and that do not
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (16, 1, 64), (8, 2, 128), (12, 1, 128), (3, 1, 40), (8, 1, 200),
                                          (10, 1, 256)])
@pytest.mark.parametrize("gap", [9, 12, 15, 17, 18, 22])
def test_attend_keeps_the_small_weights_beside_a_dominant_score(dtype, heads, kv, dim, gap):
    """One key's score is far above the others' and its value is zero, as with
    an attention sink: the result is what the others' small weights leave.

    The scores are exact (one product each, of whole numbers).  A weight's
    numerator is off by 8 u relatively and by 2^-16 (two bf16 terms), or by
    2^-21 and, absolutely, 2^-40 of the largest (two fp16 terms): over n keys
    n 2^-40 max |v| / l, with l >= 1.  Sums over n rows as tensor cores add them:
    (n + 24) 4 u, of numerator and denominator.
    """
    for n in (33, 8192):
        rng = np.random.default_rng(n + gap)
        c = Cache(rng, [n], kv, dim, 16, dtype)
        _sink(c, gap, torch.from_numpy(rng.uniform(100, 1000, (kv, n, dim)).astype(np.float32)))
        q = torch.zeros(1, heads, dim, dtype=T[dtype])
        q[:, :, 0] = 1
        q = q.cuda()
        h = c.handle(heads)
        out = h.attend(c.k, c.v, q, c.table, c.lengths(), torch.empty_like(q), scale=1.0)
        h.synchronize()
        ref, mag, _, _ = _reference(q[0].cpu(), c.rows[0][0], c.rows[0][1], 1.0, None)
        terms, floor = (2.0 ** -21, 2.0 ** -40) if dtype == "f16" else (2.0 ** -16, 0.0)
        rel = 2 * ((n + 24) * 4 * U + terms)
        tol = rel * mag + n * floor * 1000 + _half_step(dtype) * (1 + rel) * np.abs(ref)
        if dtype == "f16":
            tol = tol + 2.0 ** -25  # half the smallest step of fp16
        err = np.abs(out[0].cpu().double().numpy() - ref)
        assert (err <= tol).all(), f"{n} rows: off by {err.max():.3e} of {np.abs(ref).max():.3e}, {(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (24, 2, 128), (8, 1, 200)])
def test_attend_large_fp16_scores(heads, kv, dim):
    """Scores of some hundreds, of both signs, in fp16: the running maximum moves by far."""
    c = Cache(np.random.default_rng(6), [500, 37, 1025], kv, dim, 16, "f16")
    _run(c, heads, "f16", q_scale=60.0)
    _run(c, heads, "f16", q_scale=60.0, scale=-0.125)
    _run(c, heads, "f16", scale=0.0)


# (pages, activations), heads, kv heads, head dim: fp32 lanes of one and two keys, of 4 to 32 lanes a row, and tensor cores
FORMS = [("f32", "f32", 3, 3, 24), ("f32", "f32", 9, 3, 64), ("f32", "f32", 8, 1, 128), ("f32", "f32", 7, 1, 200),
         ("bf16", "f32", 4, 1, 200), ("f16", "f32", 6, 2, 48), ("bf16", "bf16", 4, 2, 8), ("f16", "f16", 4, 2, 64),
         ("bf16", "bf16", 16, 1, 64), ("bf16", "bf16", 8, 2, 128), ("f16", "f16", 12, 1, 96), ("bf16", "bf16", 8, 1, 256)]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_queries_that_are_not_finite_leave_masked_rows_out(form, value):
    """Sequences whose rows are all taken out give zeros and no weights whatever
    their queries hold, as the unused rows of a padded batch do; beside
    attended rows such a query spoils its own head only."""
    cache, act, heads, kv, dim = form
    rng = np.random.default_rng(90)
    lens = [3, 600, 70, 0, 90]
    c = Cache(rng, lens, kv, dim, 16, cache)
    n = c.cols * c.page
    mask = torch.zeros(5, n)
    mask[:2] = -float("inf")
    mask[2, :40] = -float("inf")
    q = _normal(rng, (5, heads, dim), act)
    q[0] = q[3] = value
    q[1, :, 1] = value
    q[2, heads - 1, 2] = value
    q, mask = q.cuda(), mask.cuda()
    w = torch.rand((5, kv, n), device="cuda")
    wo = torch.full_like(w, 5.0)
    h = c.handle(heads, weights=True)
    out = h.attend(c.k, c.v, q, c.table, c.lengths(), torch.full_like(q, 7.0), mask=mask, weights=w, weights_out=wo)
    h.synchronize()
    for i in (0, 1, 3):
        assert (out[i] == 0).all(), f"sequence {i}"
        assert torch.equal(wo[i, :, :lens[i]], w[i, :, :lens[i]])
    assert not torch.isfinite(out[2, heads - 1].float()).all()
    assert torch.isfinite(out[2, :heads - 1].float()).all() and torch.isfinite(out[4].float()).all()
    assert torch.equal(wo[2, :, :40], w[2, :, :40])
    c.lens = [-1, -1, -1, -1, 90]
    out[:4] = 7
    wo[:4] = 5
    before = torch.full_like(w, 5.0)
    _check_attend(c, q, out, act, dim ** -0.5, None, w, wo, before)


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_mask_value_of_nan_or_infinity_gives_nan(form, value):
    """In its own sequence only, wherever it lies: in the first, a middle or the last row of one or of many tiles."""
    cache, act, heads, kv, dim = form
    rng = np.random.default_rng(91)
    lens = [1, 700, 30, 2500, 45]
    c = Cache(rng, lens, kv, dim, 16, cache)
    n = c.cols * c.page
    mask = torch.zeros(5, n)
    for i, at in ((0, 0), (1, 0), (2, 17), (3, 2499)):
        mask[i, at] = value
    mask[2, :17] = -float("inf")
    q = _normal(rng, (5, heads, dim), act).cuda()
    h = c.handle(heads, weights=True)
    wo = torch.full((5, kv, n), 5.0, device="cuda")
    before = wo.clone()
    out = h.attend(c.k, c.v, q, c.table, c.lengths(), torch.full_like(q, 7.0), mask=mask.cuda(), weights_out=wo)
    h.synchronize()
    assert torch.isnan(out[:4].float()).all()
    out[:4] = 7
    wo[:4] = 5
    c.lens = [-1, -1, -1, -1, 45]
    _check_attend(c, q, out, act, dim ** -0.5, None, None, wo, before)


def test_evictions_that_overlap_on_one_handle_spoil_no_later_one():
    """Two streams without an order, one handle: lengths and budgets differ, so
    that each call may find the other's plan.  Their own results are lost; what
    lies around their arrays, and the calls after them, are not."""
    rng = np.random.default_rng(92)
    kv, dim, page, batch = 2, 16, 16, 6

    def case(lens, budget, seed):
        c = Cache(np.random.default_rng(seed), lens, kv, dim, page, "bf16")
        n = c.cols * page
        around = torch.full((batch * kv * n + 64,), 3.0, device="cuda")  # weights with a margin on both sides
        w = around[32:-32].view(batch, kv, n)
        w.copy_(torch.from_numpy(rng.random((batch, kv, n), dtype=np.float32)))
        kept = torch.full((batch * kv * budget + 64,), 55, dtype=torch.int32, device="cuda")
        return dict(c=c, w=w, lens=c.lengths(), budget=budget, kept=kept[32:-32].view(batch, kv, budget), around=around,
                    kept_around=kept, lens_out=torch.zeros(batch, dtype=torch.int32, device="cuda"))

    def evict(h, x, stream=None):
        h.evict(x["c"].k, x["c"].v, x["w"], x["c"].table, x["lens"], x["budget"], 5, x["kept"], x["w"], x["lens_out"],
                stream=stream)

    few, many = [1, 0, 3, -1, 2, 5], [900, 700, 33, 2000, -1, 1500]
    cases = [case(few, 400, 1), case(many, 40, 2)]
    cases[0]["c"].num_pages = cases[1]["c"].num_pages = max(x["c"].num_pages for x in cases)
    for x in cases:  # pages of one shape, for one handle
        for name in ("k", "v"):
            p = torch.zeros((x["c"].num_pages,) + getattr(x["c"], name).shape[1:], dtype=torch.bfloat16, device="cuda")
            p[:getattr(x["c"], name).shape[0]] = getattr(x["c"], name)
            setattr(x["c"], name, p)
    h = cases[1]["c"].handle(kv, max_pages=200)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(40):
        for x, s in zip(cases, streams):
            evict(h, x, s)
    torch.cuda.synchronize()
    try:
        h.synchronize()  # a spoilt call may have found a position without a page
    except Exception as e:
        assert "device reported" in str(e)
    for x in cases:
        for margin, value in ((x["around"], 3), (x["kept_around"], 55)):
            assert (margin[:32] == value).all() and (margin[-32:] == value).all()
    # the same handle again, in order, and a new one
    again, fresh = case(many, 40, 3), case(many, 40, 3)
    fresh["w"].copy_(again["w"])
    h2 = fresh["c"].handle(kv, max_pages=200)
    assert again["c"].num_pages == cases[1]["c"].num_pages
    evict(h, again)
    evict(h2, fresh)
    h.synchronize()
    h2.synchronize()
    for name in ("kept", "w", "lens_out"):
        assert torch.equal(again[name], fresh[name]), name
    assert torch.equal(torch.nan_to_num(again["c"].k), torch.nan_to_num(fresh["c"].k))
    assert again["lens_out"].tolist() == [40, 40, 33, 40, -1, 40]


@pytest.mark.parametrize("form", [("f32", "f32", 8, 1, 200), ("f32", "f32", 14, 2, 256), ("bf16", "f32", 4, 1, 200),
                                  ("f16", "f32", 8, 2, 256), ("f32", "bf16", 6, 1, 136)], ids=lambda f: "-".join(map(str, f)))
def test_long_rows_give_the_same_bits_again(form):
    """Rows of more than 128 elements, whose partial sums take the place of the
    values that the last tile of a segment held: many segments of a few tiles."""
    cache, act, heads, kv, dim = form
    rng = np.random.default_rng(93)
    c = Cache(rng, [int(x) for x in rng.integers(1, 150, 120)], kv, dim, 16, cache)
    h = c.handle(heads)
    first = _run(c, heads, act, kv=h)
    q = _normal(np.random.default_rng(3), (120, heads, dim), act, 2.0).cuda()
    outs = [h.attend(c.k, c.v, q, c.table, c.lengths(), torch.empty_like(q)) for _ in range(10)]
    h.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")],
                         ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("group", [1, 3, 5, 11])
def test_every_head_dim(types, group):
    """All multiples of 8 up to 256, the new row stored and weights added: ends inside and at the end of tiles and pages."""
    for dim in range(8, 257, 8):
        c = Cache(np.random.default_rng(dim), [1, 31, 32, 140, 65], 2, dim, (16, 7, 33)[dim // 8 % 3], types[0])
        _run(c, 2 * group, types[1], seed=dim + group, new=True, with_weights=True)


@pytest.mark.parametrize("types,dim", [(("bf16", "bf16"), 16), (("f16", "f16"), 64), (("f32", "f32"), 8), (("bf16", "f32"), 8)],
                         ids=lambda v: "-".join(v) if isinstance(v, tuple) else str(v))
def test_attend_the_longest_sequence(types, dim):
    """2^31 - 2^20 - 1024 rows, whose table names one page again and again.

    Keys of zeros make every weight 1, and values of 0 and 1 every sum of a block
    a whole number below 2^24, so exact.  A sum of the blocks' parts, of at most
    592 blocks, and the division round 600 times at most: 2 * 600 u relatively.
    """
    page = 1024
    cols = (1 << 21) - 1025
    k = torch.zeros((2, 1, page, dim), dtype=T[types[0]], device="cuda")
    v = torch.full_like(k, float("nan"))
    ones = torch.arange(page)[:, None] * (torch.arange(dim)[None] + 1) % 3 == 0
    v[1, 0] = ones.cuda().to(T[types[0]])
    table = torch.ones((1, cols), dtype=torch.int32, device="cuda")
    from gawee_b200.paged_kv import PagedKV
    h = PagedKV(types[0], 2, 1, dim, page, 2, 1, cols)
    q = torch.ones((1, 2, dim), dtype=T[types[1]], device="cuda")
    lens = torch.tensor([cols * page], dtype=torch.int32, device="cuda")
    out = h.attend(k, v, q, table, lens, torch.empty_like(q))
    h.synchronize()
    want = ones.double().mean(0).expand(2, dim)
    tol = want * (1200 * U + _half_step(types[1])) + 1e-30
    err = (out[0].cpu().double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16")], ids=lambda t: f"{t[0]}-{t[1]}")
def test_the_largest_batch_and_the_largest_group(types):
    """65,535 sequences of a few rows or none; 4096 query heads over one key/value head."""
    rng = np.random.default_rng(94)
    lens = [int(x) for x in rng.choice([-1, 0, 1, 2, 9], 65535)]
    c = Cache(rng, [1], 1, 8, 4, types[0])  # one page, of which every sequence reads the first rows
    c.k.nan_to_num_(nan=0.5)
    c.v = _normal(rng, c.v.shape, types[0]).cuda()
    h = _kv(types[0], 2, 1, 8, 4, c.num_pages, max_batch=65535, max_pages=3, weights=True)
    table = torch.randint(0, c.num_pages, (65535, 3), dtype=torch.int32, device="cuda")
    q = _normal(rng, (65535, 2, 8), types[1]).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wo = torch.full((65535, 1, 12), 5.0, device="cuda")
    out = h.attend(c.k, c.v, q, table, lengths, torch.full_like(q, 7.0), weights_out=wo)
    h.synchronize()
    # the same in smaller batches, whose results the other tests hold against the formula
    small = _kv(types[0], 2, 1, 8, 4, c.num_pages, max_batch=1000, max_pages=3, weights=True)
    for at in range(0, 65535, 1000):
        part = slice(at, min(at + 1000, 65535))
        w1 = torch.full_like(wo[part], 5.0)
        o1 = small.attend(c.k, c.v, q[part], table[part], lengths[part], torch.full_like(q[part], 7.0), weights_out=w1)
        assert torch.equal(out[part], o1) and torch.equal(wo[part], w1), at
    small.synchronize()
    wide = Cache(rng, [300, 5], 1, 16, 16, types[0])
    _run(wide, 4096, types[1], with_weights=True, new=True)
