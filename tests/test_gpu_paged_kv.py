"""Paged key/value cache on the GPU against plain 64-bit implementations.

Unused rows and pages hold NaN, so that a read behind a sequence shows.

Tolerance of attend, with u = 2^-24 and worst-case bounds throughout.  A score
is a sum of D products and a few roundings (scale, mask): off by at most
ds = (D + 4) u S + 3 u |s| with S = |scale| sum_d |q_d k_d|; with a 16-bit
query and cache the products may be summed by tensor cores, which keep 22 bits
or more: 4 u in place of u.  Each weight's numerator exp(s - m) is off by
2 ds + 8 u relatively (m shifts all of them alike), and by 2^-16 more where
tensor cores take it as two bf16 terms (2^-21 as two fp16 terms, of at most
1, whose smallest step is 2^-24).  Sums over n rows add (n + 16) u.  Numerator
and denominator together: out is off by at most
    2 (2 max ds + (n + 24) a) sum_i p_i |v_i|  +  half a step of its type,
with a = u, or 4 u + 2^-16 / 2^-21 as above over the same sums, and by
A = 2^-23 max |v| for fp16 terms below its smallest step.  Weights: the same
relative bound times p, plus a rounding of the sum.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def _kv(*a, **kw):
    from gawee_b200.paged_kv import PagedKV
    return PagedKV(*a, **kw)


def _normal(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32) * np.float32(scale)).to(T[dtype])


class Cache:
    """Pages and table of sequences with the given rows; everything else is NaN or -1."""

    def __init__(self, rng, lens, kv_heads, dim, page, dtype, spare_rows=0, interleaved=False, extra_cols=2):
        self.page, self.lens, self.kv_heads, self.dim, self.dtype = page, list(lens), kv_heads, dim, dtype
        counts = [-(-(max(n, 0) + spare_rows) // page) for n in lens]
        self.cols = max(counts + [1]) + extra_cols
        self.num_pages = sum(counts) + 3
        perm = rng.permutation(self.num_pages)
        table = np.full((len(lens), self.cols), -1, np.int32)
        at = 0
        for i, c in enumerate(counts):
            table[i, :c] = perm[at:at + c]
            at += c
        self.counts, self.table_np = counts, table
        self.table = torch.from_numpy(table).cuda()
        shape = (self.num_pages, kv_heads, page, dim)
        if interleaved:
            both = torch.full((self.num_pages, 2) + shape[1:], float("nan"), dtype=T[dtype], device="cuda")
            self.k, self.v = both[:, 0], both[:, 1]
            self.page_stride = 2 * kv_heads * page * dim
        else:
            self.k, self.v = (torch.full(shape, float("nan"), dtype=T[dtype], device="cuda") for _ in range(2))
            self.page_stride = 0
        self.rows = []  # (k, v) [kv_heads, n, dim] of each sequence, cpu, of the pages' type
        for i, n in enumerate(lens):
            kk, vv = (_normal(rng, (kv_heads, max(n, 0), dim), dtype) for _ in range(2))
            self.rows.append([kk, vv])
            self.put(i)

    def put(self, i):
        for which, pages in ((0, self.k), (1, self.v)):
            r = self.rows[i][which]
            for c in range(-(-r.shape[1] // self.page)):
                part = r[:, c * self.page:(c + 1) * self.page]
                pages[int(self.table_np[i, c]), :, :part.shape[1]] = part.cuda()

    def get(self, pages, i, n):
        ids = torch.from_numpy(self.table_np[i, :-(-n // self.page)].astype(np.int64)).cuda()
        return pages[ids].transpose(0, 1).flatten(1, 2)[:, :n].cpu()

    def lengths(self):
        return torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def handle(self, heads, **kw):
        kw.setdefault("max_batch", len(self.lens))
        kw.setdefault("max_pages", self.cols)
        return _kv(self.dtype, heads, self.kv_heads, self.dim, self.page, self.num_pages,
                   page_stride=self.page_stride, **kw)


def _reference(q, k, v, scale, mask):
    """Of one sequence in 64 bits: (out, tolerance pieces, weights); k, v [kv, n, dim], q [heads, dim]."""
    heads, dim = q.shape
    kv, n = k.shape[:2]
    g = heads // kv
    out, mag, ds = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros(heads)
    p_all = np.zeros((heads, n))
    q, k, v = (x.double().numpy() for x in (q, k, v))
    live = np.ones(n, bool) if mask is None else ~np.isneginf(mask)
    for h in range(heads if live.any() else 0):
        kk, vv = k[h // g][live], v[h // g][live]
        s = kk @ q[h] * scale
        size = np.abs(kk) @ np.abs(q[h]) * abs(scale)
        if mask is not None:
            s = s + mask[live].astype(np.float64)
        # beside a mask of the lowest value a score is lost entirely, here as in fp32
        ds[h] = ((dim + 4) * U * size + 3 * U * np.where(np.abs(s) < 1e30, np.abs(s), 0.0)).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        p_all[h, live] = p
    return out, mag, ds, p_all


def _half_step(dtype):
    return torch.finfo(T[dtype]).eps / 2


def _terms(act, cache):
    """(relative error of an addition or of a weight's terms, of a score's, absolute of a weight) by the types."""
    if act == cache == "bf16":
        return 4 * U, 2.0 ** -16, 4, 0.0
    if act == cache == "f16":
        return 4 * U, 2.0 ** -21, 4, 2.0 ** -23
    return U, 0.0, 1, 0.0


def _check_attend(c, q, out, act, scale, mask, weights=None, weights_out=None, before=None):
    """Compare a call's results with the reference, row by row."""
    heads = q.shape[1]
    g = heads // c.kv_heads
    out, q = out.cpu(), q.cpu()
    add, terms, wide, absolute = _terms(act, c.dtype)
    for i, n in enumerate(c.lens):
        if n < 0:
            assert torch.equal(out[i].float(), torch.full_like(out[i], 7.0).float()), f"row {i} of no sequence was written"
            if weights_out is not None:
                assert torch.equal(weights_out[i].cpu(), before[i].cpu())
            continue
        m = None if mask is None else mask[i if mask.shape[0] > 1 else 0, :n].cpu().numpy()
        ref, mag, ds, p = _reference(q[i], c.rows[i][0][:, :n], c.rows[i][1][:, :n], scale, m)
        rel = 2 * (2 * wide * ds[:, None] + (n + 24) * add + terms)
        vmax = float(np.nanmax(np.abs(ref)) if n == 0 else np.nan_to_num(c.rows[i][1][:, :n].double().abs().numpy(), posinf=0).max())
        tol = rel * mag + absolute * vmax + _half_step(act) * (1 + rel) * np.abs(ref) + 1e-30
        if act == "f16":
            tol = tol + 2.0 ** -25  # half the smallest step of fp16
        err = np.abs(out[i].double().numpy() - ref)
        assert (err <= tol).all(), f"sequence {i} of {n} rows: off by {err.max():.3e}, {(err / tol).max():.2f} of the tolerance"
        if weights_out is not None:
            w = np.zeros((c.kv_heads, n)) if weights is None else weights[i, :, :n].cpu().double().numpy()
            step = p.reshape(c.kv_heads, g, n)
            want = w + step.sum(1)
            tol = (step * rel.reshape(c.kv_heads, g, 1)).sum(1) + (g + 2) * U * np.abs(want) + 1e-30
            err = np.abs(weights_out[i, :, :n].cpu().double().numpy() - want)
            assert (err <= tol).all(), f"weights of {i}: off by {err.max():.3e}, {(err / tol).max():.2f} of the tolerance"
            assert torch.equal(weights_out[i, :, n:].cpu(), before[i, :, n:].cpu()), "columns behind the length were written"


def _run(c, heads, act, seed=3, mask=None, with_weights=False, weights_in_place=False, new=False, scale=None, kv=None,
         stream=None, q_scale=2.0):
    rng = np.random.default_rng(seed)
    batch = len(c.lens)
    q = _normal(rng, (batch, heads, c.dim), act, q_scale).cuda()
    out = torch.full_like(q, 7.0)
    w = wo = before = None
    n = c.cols * c.page
    if with_weights:
        w = torch.from_numpy(rng.random((batch, c.kv_heads, n), dtype=np.float32)).cuda()
        wo = w if weights_in_place else torch.full_like(w, 5.0)
        before = wo.clone()
    first = None if w is None else w.clone()
    k = v = None
    if new:
        k, v = (_normal(rng, (batch, c.kv_heads, c.dim), act).cuda() for _ in range(2))
        for i, ln in enumerate(c.lens):
            if ln > 0:
                for which, x in ((0, k), (1, v)):
                    c.rows[i][which][:, ln - 1] = x[i].cpu().to(T[c.dtype])
    h = kv or c.handle(heads, weights=with_weights)
    pages_before = (c.k.clone(), c.v.clone())
    used = scale if scale is not None else c.dim ** -0.5
    got = h.attend(c.k, c.v, q, c.table, c.lengths(), out, scale=scale, k=k, v=v, mask=mask, weights=w, weights_out=wo,
                   stream=stream)
    h.synchronize(stream)
    assert got is out
    _check_attend(c, q, out, act, used, mask, first, wo, before)
    for which, pages in ((0, c.k), (1, c.v)):
        want = pages_before[which]
        if new:
            for i, ln in enumerate(c.lens):
                if ln > 0:
                    want[int(c.table_np[i, (ln - 1) // c.page]), :, (ln - 1) % c.page] = \
                        c.rows[i][which][:, ln - 1].to(want)
        assert torch.equal(torch.nan_to_num(pages.float(), nan=123.0), torch.nan_to_num(want.float(), nan=123.0)), \
            "pages were changed"
    return out


# (pages, activations), query heads over key/value heads, head dim, page size
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32"), ("f32", "bf16"), ("f16", "bf16")]
SHAPES = [(6, 6, 48, 16), (9, 3, 64, 16), (8, 1, 128, 64), (15, 5, 80, 24), (4, 2, 8, 1), (12, 1, 256, 7), (32, 2, 96, 100),
          (7, 1, 200, 32), (20, 10, 40, 8)]
LENS = [1, 0, 5, 130, 16, 17, -1, 64, 301, 15, 33, 128]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attend(types, shape):
    heads, kv, dim, page = shape
    c = Cache(np.random.default_rng(1), LENS, kv, dim, page, types[0])
    _run(c, heads, types[1])


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("shape", SHAPES[:6], ids=lambda s: "x".join(map(str, s)))
def test_attend_stores_the_new_row_and_adds_weights(types, shape):
    heads, kv, dim, page = shape
    c = Cache(np.random.default_rng(2), LENS, kv, dim, page, types[0], interleaved=True)
    _run(c, heads, types[1], with_weights=True, new=True)
    _run(c, heads, types[1], with_weights=True, weights_in_place=True, seed=4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (4, 2), (8, 2), (9, 1), (16, 1), (33, 1), (64, 4)])
def test_attend_group_sizes(dtype, heads, kv):
    c = Cache(np.random.default_rng(3), [70, 1, 257], kv, 64, 16, dtype)
    _run(c, heads, dtype, new=True, with_weights=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [2000], [4097, 3], [1] * 70, [0, 0], [-1, -1, -1], [0, -1, 900], [511] * 9],
                         ids=lambda v: f"{len(v)}x{v[0]}")
def test_attend_lengths(dtype, lens):
    c = Cache(np.random.default_rng(4), lens, 2, 64, 16, dtype)
    _run(c, 6, dtype)
    _run(c, 6, dtype, with_weights=True, seed=8)


@pytest.mark.parametrize("types", TYPES[:4], ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("kind", ["padding", "nothing", "lowest", "bias", "shared", "holes"])
def test_attend_masks(types, kind):
    rng = np.random.default_rng(5)
    c = Cache(rng, [40, 200, 1, 0, 333, 64], 2, 64, 16, types[0])
    n = c.cols * c.page
    mask = np.zeros((6, n), np.float32)
    if kind == "padding":
        for i, ln in enumerate(c.lens):
            mask[i, :ln // 3] = -np.inf
    elif kind == "nothing":  # rows 0 and 4 attend to nothing
        mask[0] = mask[4] = -np.inf
    elif kind == "lowest":  # a whole row of the lowest value: still a softmax over its rows
        mask[1] = np.finfo(np.float32).min
        mask[4, 7:] = np.finfo(np.float32).min
    elif kind == "bias":
        mask[:] = rng.standard_normal(mask.shape)
    elif kind == "shared":
        mask = np.where(rng.random((1, n)) < 0.5, -np.inf, 0.0).astype(np.float32)
    else:
        mask[rng.random(mask.shape) < 0.9] = -np.inf
        mask[4, :300] = -np.inf
    # rows that the mask takes out may hold anything
    m = np.broadcast_to(mask, (6, n))
    for i, ln in enumerate(c.lens):
        dead = torch.from_numpy(np.isneginf(m[i, :ln]).copy())
        for which in (0, 1):
            c.rows[i][which][:, dead] = float("nan")
            if dead.any():
                c.rows[i][which][:, int(dead.nonzero()[0])] = float("inf")
        c.put(i)
    for i, ln in enumerate(c.lens):  # the reference drops them by the mask
        for which in (0, 1):
            c.rows[i][which] = torch.nan_to_num(c.rows[i][which], nan=0.0, posinf=0.0)
    _run(c, 6, types[1], mask=torch.from_numpy(mask).cuda(), with_weights=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_large_scores(dtype):
    """Scores of some hundreds, of both signs: the running maximum moves by far."""
    c = Cache(np.random.default_rng(6), [500, 37, 1025], 2, 64, 16, dtype)
    _run(c, 4, dtype, q_scale=60.0)
    _run(c, 4, dtype, q_scale=60.0, scale=-0.125)
    _run(c, 4, dtype, scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_nan_in_attended_rows_stays_in_its_sequence_and_head(dtype):
    c = Cache(np.random.default_rng(7), [50, 60], 2, 64, 16, dtype)
    c.k[int(c.table_np[0, 1]), 1, 3] = float("nan")
    q = _normal(np.random.default_rng(1), (2, 4, 64), dtype).cuda()
    out = c.handle(4).attend(c.k, c.v, q, c.table, c.lengths(), torch.empty_like(q), stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    bad = torch.isnan(out.float()).flatten(2).any(-1).cpu()
    assert bad.tolist() == [[False, False, True, True], [False] * 4]


def test_attend_strides_of_wider_arrays_and_a_larger_table():
    rng = np.random.default_rng(8)
    c = Cache(rng, [100, 3, 250], 3, 64, 16, "f32", interleaved=True)
    heads, n = 9, c.cols * c.page
    qkv = torch.from_numpy(rng.standard_normal((3, 15 * 64 + 5), dtype=np.float32)).cuda()
    q = qkv.as_strided((3, 9, 64), (965, 64, 1), 1)
    k = qkv.as_strided((3, 3, 64), (965, 64, 1), 1 + 9 * 64)
    v = qkv.as_strided((3, 3, 64), (965, 64, 1), 1 + 12 * 64)
    wide = torch.full((3, 20, 64), 7.0, device="cuda")
    out = wide[:, 2:11]
    table = torch.full((3, c.cols + 9), -5, dtype=torch.int32, device="cuda")
    table[:, :c.cols] = c.table
    mask = torch.zeros((3, n + 13), device="cuda")[:, 5:5 + n]
    w = torch.zeros((3, 3, n + 3), device="cuda")[:, :, 1:1 + n]
    wo = torch.full((3, 7, n), 5.0, device="cuda")[:, 2:5]
    before = wo.clone()
    for i, ln in enumerate(c.lens):
        c.rows[i][0][:, ln - 1], c.rows[i][1][:, ln - 1] = k[i].cpu(), v[i].cpu()
    h = c.handle(heads, weights=True, max_pages=c.cols + 4, max_batch=9)
    h.attend(c.k, c.v, q, table[:, :c.cols], c.lengths(), out, k=k, v=v, mask=mask, weights=w, weights_out=wo)
    h.synchronize()
    _check_attend(c, q, out, "f32", 0.125, mask, w, wo, before)
    assert (wide[:, :2] == 7).all() and (wide[:, 11:] == 7).all()


def test_attend_beyond_32_bit_offsets():
    """Pages whose elements pass 2^31: the first, one in the middle and the last."""
    pages, kv, page, dim = 2100, 8, 1024, 128
    k, v = (torch.empty((pages, kv, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 31
    c = Cache(np.random.default_rng(9), [2500], kv, dim, page, "bf16")
    big = [pages - 1, 7, 2048]
    for i in range(3):
        k[big[i]], v[big[i]] = c.k[int(c.table_np[0, i])], c.v[int(c.table_np[0, i])]
    c.k, c.v, c.num_pages = k, v, pages
    c.table_np[0, :3] = big
    c.table = torch.from_numpy(c.table_np).cuda()
    q = _normal(np.random.default_rng(2), (1, 16, dim), "bf16").cuda()
    h = c.handle(16)
    out = h.attend(k, v, q, c.table, c.lengths(), torch.empty_like(q))
    h.synchronize()
    _check_attend(c, q, out, "bf16", dim ** -0.5, None)
    row = torch.full((1, kv, dim), 3.0, device="cuda")
    h.append(k, v, row, row, c.table, torch.tensor([5], dtype=torch.int32, device="cuda"))
    h.synchronize()
    assert (k[pages - 1, :, 5] == 3).all() and (v[pages - 1, :, 5] == 3).all()


def test_attend_gives_the_same_bits_again():
    for dtype in ("f32", "bf16"):
        c = Cache(np.random.default_rng(10), [3000, 17, 900, 4000], 2, 128, 16, dtype)
        q = _normal(np.random.default_rng(3), (4, 16, 128), dtype).cuda()
        h = c.handle(16, weights=True)
        w = torch.zeros((4, 2, c.cols * c.page), device="cuda")
        outs = []
        for _ in range(20):
            wo = torch.zeros_like(w)
            outs.append((h.attend(c.k, c.v, q, c.table, c.lengths(), torch.empty_like(q), weights=w, weights_out=wo), wo))
        h.synchronize()
        assert all(torch.equal(o, outs[0][0]) and torch.equal(x, outs[0][1]) for o, x in outs)


def test_captured_step_follows_the_lengths_and_shares_the_handle():
    """One graph per layer over one handle, replayed in order on a stream, while
    the lengths grow on the device; then eager calls again."""
    rng = np.random.default_rng(11)
    layers = [Cache(rng, [20, 1, 130], 3, 64, 16, "f32", spare_rows=40) for _ in range(2)]
    h = layers[0].handle(9, weights=False, max_pages=16)
    big = max(c.num_pages for c in layers)
    assert all(c.num_pages == big for c in layers)
    s = torch.cuda.Stream()
    lens = torch.tensor([20, 1, 130], dtype=torch.int32, device="cuda")
    io = []
    graphs = []
    with torch.cuda.stream(s):
        for c in layers:
            q, k, v = (torch.zeros((3, n, 64), device="cuda") for n in (9, 3, 3))
            out = torch.zeros_like(q)
            h.attend(c.k, c.v, q, c.table, lens, out, k=k, v=v, stream=s)
            io.append((q, k, v, out))
        s.synchronize()
        for c, (q, k, v, out) in zip(layers, io):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                h.attend(c.k, c.v, q, c.table, lens, out, k=k, v=v, stream=torch.cuda.current_stream())
            graphs.append(g)
        for step in range(1, 36):
            lens += 1
            for c, (q, k, v, out), g in zip(layers, io, graphs):
                q.copy_(_normal(rng, (3, 9, 64), "f32"))
                k.copy_(_normal(rng, (3, 3, 64), "f32"))
                v.copy_(_normal(rng, (3, 3, 64), "f32"))
                g.replay()
                for i in range(3):
                    for which, x in ((0, k), (1, v)):
                        c.rows[i][which] = torch.cat([c.rows[i][which], x[i].cpu()[:, None]], 1)
                c.lens = [n + 1 for n in c.lens]
                if step % 7 == 0:
                    h.synchronize(s)
                    # the first row was overwritten by the call before the capture (zeros at row length - 1)
                    for i, n0 in enumerate([20, 1, 130]):
                        c.rows[i][0][:, n0 - 1] = 0
                        c.rows[i][1][:, n0 - 1] = 0
                    _check_attend(c, q, out, "f32", 0.125, None)
    h.synchronize(s)


def test_calls_on_two_streams_ordered_by_events():
    c = Cache(np.random.default_rng(12), [700, 90], 2, 64, 16, "bf16")
    h = c.handle(8)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    q = _normal(np.random.default_rng(1), (2, 8, 64), "bf16").cuda()
    torch.cuda.synchronize()
    outs = []
    for i in range(10):
        s = (a, b)[i % 2]
        s.wait_stream((b, a)[i % 2])
        outs.append(torch.empty_like(q))
        h.attend(c.k, c.v, q, c.table, c.lengths(), outs[-1], stream=s)
        torch.cuda.synchronize() if i == 0 else None
    h.synchronize(a)
    h.synchronize(b)
    for o in outs:
        _check_attend(c, q, o, "bf16", 0.125, None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["page", "negative", "length", "mask", "weights"])
def test_what_only_the_device_sees_is_reported_and_touches_nothing(dtype, what):
    from gawee_b200.runtime import GaweeError
    c = Cache(np.random.default_rng(13), [40, 100, 60], 2, 64, 16, dtype)
    h = c.handle(4, weights=True)
    q = _normal(np.random.default_rng(1), (3, 4, 64), dtype).cuda()
    out = torch.full_like(q, 7.0)
    lens, kw, text = c.lengths(), {}, "sequence longer"
    n = c.cols * c.page
    if what in ("page", "negative"):
        c.table[1, 3] = c.num_pages if what == "page" else -3
        text = "block table"
    elif what == "length":
        lens[1] = n + 1
    elif what == "mask":
        kw["mask"] = torch.zeros((3, 99), device="cuda")
    else:
        kw["weights_out"] = torch.zeros((3, 2, 99), device="cuda")
    k = _normal(np.random.default_rng(2), (3, 2, 64), dtype).cuda()
    pages = c.k.clone()
    h.attend(c.k, c.v, q, c.table, lens, out, k=k, v=k, **kw)
    with pytest.raises(GaweeError, match=text) as e:
        h.synchronize()
    assert e.value.status == 6
    h.synchronize()  # the word is cleared
    if what not in ("page", "negative"):
        assert (out[1] == 0).all()
        assert torch.equal(torch.nan_to_num(c.get(c.k, 1, 100).float()), torch.nan_to_num(c.get(pages, 1, 100).float()))
    for i in (0, 2):
        for which in (0, 1):
            c.rows[i][which][:, c.lens[i] - 1] = k[i].cpu()
    c.lens[1] = 0
    out[1] = 0
    _check_attend(c, q, out, dtype, 0.125, None)


# --- append -------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES + [("f32", "f16"), ("bf16", "f16")], ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("kv,dim,page", [(3, 64, 16), (1, 8, 1), (5, 40, 7), (2, 256, 100), (7, 72, 3)])
def test_append(types, kv, dim, page):
    rng = np.random.default_rng(20)
    c = Cache(rng, [10, 0, 33, 5], kv, dim, page, types[0], spare_rows=30, interleaved=True)
    new = [(0, 10 + j) for j in range(25)] + [(1, j) for j in range(7)] + [(3, 5)] + [(2, 62), (2, 33)]
    new += [(-1, 4), (0, -1), (-7, -7)]  # left out
    order = rng.permutation(len(new))
    new = [new[i] for i in order]
    t = len(new)
    k = _normal(rng, (t, kv + 1, dim), types[1], 3.0).cuda()[:, 1:]
    v = _normal(rng, (t, kv, dim), types[1], 3.0).cuda()
    want = [c.k.clone(), c.v.clone()]
    for j, (b, p) in enumerate(new):
        if b >= 0 and p >= 0:
            want[0][int(c.table_np[b, p // page]), :, p % page] = k[j].to(T[types[0]])
            want[1][int(c.table_np[b, p // page]), :, p % page] = v[j].to(T[types[0]])
    h = c.handle(kv)
    seq, pos = (torch.tensor([x[i] for x in new], dtype=torch.int32, device="cuda") for i in (0, 1))
    h.append(c.k, c.v, k, v, c.table, pos, sequences=seq)
    h.synchronize()
    for got, w in zip((c.k, c.v), want):
        assert torch.equal(torch.nan_to_num(got.float(), nan=99.0), torch.nan_to_num(w.float(), nan=99.0))


@pytest.mark.parametrize("dim,offset", [(64, 0), (64, 1), (48, 2), (8, 3)])
def test_append_one_token_per_sequence_from_any_alignment(dim, offset):
    rng = np.random.default_rng(21)
    c = Cache(rng, [3, 100, 16], 3, dim, 16, "bf16", spare_rows=1)
    flat = _normal(rng, (offset + 3 * (9 * dim + 1),), "bf16").cuda()
    k = flat.as_strided((3, 3, dim), (9 * dim + 1, dim, 1), offset)
    v = flat.as_strided((3, 3, dim), (9 * dim + 1, dim, 1), offset + 3 * dim)
    h = c.handle(3)
    h.append(c.k, c.v, k, v, c.table, c.lengths())
    h.synchronize()
    for i, n in enumerate(c.lens):
        for pages, x, which in ((c.k, k, 0), (c.v, v, 1)):
            got = c.get(pages, i, n + 1)
            assert torch.equal(got[:, n], x[i].cpu()) and torch.equal(got[:, :n], c.rows[i][which])


def test_append_reports_what_it_cannot_store():
    from gawee_b200.runtime import GaweeError
    c = Cache(np.random.default_rng(22), [3, 5], 2, 64, 16, "f32")
    h = c.handle(2)
    k = torch.zeros((1, 2, 64), device="cuda")
    for seq, pos, text in ((0, 16, "block table"), (1, c.cols * 16, "block table"), (2, 0, "outside the batch"),
                           (0, (1 << 31) - 1, "block table")):
        before = c.k.clone()
        h.append(c.k, c.v, k, k, c.table, torch.tensor([pos], dtype=torch.int32, device="cuda"),
                 sequences=torch.tensor([seq], dtype=torch.int32, device="cuda"))
        with pytest.raises(GaweeError, match=text):
            h.synchronize()
        assert torch.equal(torch.nan_to_num(c.k), torch.nan_to_num(before))


def test_append_rounds_to_nearest():
    c = Cache(np.random.default_rng(23), [0], 1, 8, 1, "bf16", spare_rows=2)
    x = torch.tensor([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -1 - 2.0 ** -8, 3.4e38, float("inf"), float("nan"), -0.0, 1e-45])
    k = x.view(1, 1, 8).cuda()
    h = c.handle(1)
    h.append(c.k, c.v, k, k, c.table, torch.tensor([0], dtype=torch.int32, device="cuda"))
    h.synchronize()
    got, want = c.get(c.k, 0, 1)[0, 0].float(), x.to(torch.bfloat16).float()
    assert torch.equal(torch.nan_to_num(got, nan=5.0), torch.nan_to_num(want, nan=5.0))
    assert math.copysign(1, got[6].item()) == -1


# --- evict --------------------------------------------------------------------

def _kept(w, n, budget, recent):
    """Positions that stay, by the definition; w: numpy f32 [n]."""
    if n <= budget:
        return list(range(max(n, 0)))
    key = np.where(np.isnan(w[:n - recent]), -np.inf, w[:n - recent].astype(np.float64))
    nan = np.isnan(w[:n - recent])
    order = sorted(range(n - recent), key=lambda i: (nan[i], -key[i], i))
    return sorted(order[:budget - recent]) + list(range(n - recent, n))


WEIGHTS = {
    "random": lambda r, s: r.random(s, dtype=np.float32) ** 8,
    "ties": lambda r, s: r.integers(0, 3, s).astype(np.float32),
    "equal": lambda r, s: np.ones(s, np.float32),
    "zeros": lambda r, s: np.where(r.random(s) < 0.5, np.float32(0.0), np.float32(-0.0)),
    "wide": lambda r, s: (r.standard_normal(s) * 10.0 ** r.integers(-44, 38, s)).astype(np.float32),
    "odd": lambda r, s: r.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, 0, 1, -1, 1e-45], np.float32), s),
    "falling": lambda r, s: np.broadcast_to(-np.arange(s[-1], dtype=np.float32), s).copy(),
    "rising": lambda r, s: np.broadcast_to(np.arange(s[-1], dtype=np.float32), s).copy(),
}


def _evict(lens, kv, dim, page, dtype, budget, recent, kind, in_place, seed=30, alias=False, runs=1):
    rng = np.random.default_rng(seed)
    c = Cache(rng, lens, kv, dim, page, dtype, interleaved=not in_place)
    batch, n = len(lens), c.cols * page
    w = WEIGHTS[kind](rng, (batch, kv, n))
    weights = torch.from_numpy(w).cuda()
    wo = weights if alias else torch.full_like(weights, 5.0)
    before = wo.cpu().clone()
    lengths = c.lengths()
    lo = lengths if alias else torch.full_like(lengths, 77)
    kept = torch.full((batch, kv, budget), 55, dtype=torch.int32, device="cuda")
    to = None
    to_np = c.table_np
    pages = [c.k, c.v]
    if not in_place:
        counts = [-(-max(0, min(x, budget)) // page) for x in lens]
        more = torch.full((c.num_pages + sum(counts), 2, kv, page, dim), float("nan"), dtype=T[dtype], device="cuda")
        more[:c.num_pages, 0], more[:c.num_pages, 1] = c.k, c.v
        to_np = np.full((batch, max(counts + [1]) + 1), -1, np.int32)
        at = c.num_pages
        for i, x in enumerate(counts):
            to_np[i, :x] = np.arange(at, at + x)[::-1]
            at += x
        c.num_pages += sum(counts)
        pages = [more[:, 0], more[:, 1]]
        to = torch.from_numpy(to_np).cuda()
    start = [p.clone() for p in pages]
    h = c.handle(kv, max_pages=max(c.cols, to_np.shape[1]))
    h.evict(pages[0], pages[1], weights, c.table, lengths, budget, recent, kept, wo, lo, to_table=to)
    h.synchronize()
    got_kept, got_w, got_len = kept.cpu().numpy(), wo.cpu(), lo.cpu().tolist()
    want = [p.clone() for p in start]
    free = torch.zeros((c.num_pages, page), dtype=torch.bool)  # rows behind the budget: anything
    for i, ln in enumerate(lens):
        m = min(ln, budget)
        assert got_len[i] == (m if ln >= 0 else ln)
        for j in range(kv):
            keep = _kept(w[i, j], ln, budget, recent)
            assert got_kept[i, j].tolist() == keep + [-1] * (budget - len(keep)), (i, j, ln)
            ww = before[i, j].clone()
            if ln > 0:
                ww[:ln] = 0
                ww[:m] = torch.from_numpy(w[i, j][keep])
            assert torch.equal(torch.nan_to_num(got_w[i, j], nan=99.0), torch.nan_to_num(ww, nan=99.0))
            for which in (0, 1):
                for r, src in enumerate(keep):
                    want[which][int(to_np[i, r // page]), j, r % page] = c.rows[i][which][j, src].cuda()
        if in_place and ln > budget:
            for r in range(budget, ln):
                free[int(c.table_np[i, r // page]), r % page] = True
    live = ~free.cuda()
    for a, b in zip(pages, want):
        a, b = (torch.nan_to_num(x.float(), nan=99.0).transpose(1, 2)[live] for x in (a, b))
        assert torch.equal(a, b)


@pytest.mark.parametrize("in_place", [False, True], ids=["copied", "in_place"])
@pytest.mark.parametrize("kind", sorted(WEIGHTS))
def test_evict_weights(kind, in_place):
    _evict([200, 64, 65, 0, 1, -1, 130], 2, 16, 16, "f32", 64, 16, kind, in_place, alias=in_place)


@pytest.mark.parametrize("in_place", [False, True], ids=["copied", "in_place"])
@pytest.mark.parametrize("dtype,kv,dim,page", [("f32", 3, 64, 16), ("bf16", 8, 128, 64), ("f16", 1, 8, 1), ("bf16", 2, 40, 7),
                                               ("f32", 1, 256, 100), ("f16", 5, 200, 24)])
def test_evict_shapes(dtype, kv, dim, page, in_place):
    _evict([333, 100, 17, 600], kv, dim, page, dtype, 99, 10, "random", in_place)


@pytest.mark.parametrize("in_place", [False, True], ids=["copied", "in_place"])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (50, 50), (50, 0), (1000, 7), (1025, 1024), (3000, 100), (5000, 5000)])
def test_evict_budgets(budget, recent, in_place):
    _evict([3001, 1024, 1026, 40, 2048], 1, 8, 32, "bf16", budget, recent, "random", in_place, alias=not in_place)


def test_evict_long_sequence():
    _evict([70001], 1, 8, 256, "f32", 33333, 1111, "ties", True, alias=True)
    _evict([70001], 1, 8, 256, "f32", 33333, 1111, "wide", False)


@pytest.mark.parametrize("in_place", [False, True], ids=["copied", "in_place"])
def test_evict_reports_bad_pages_and_lengths(in_place):
    from gawee_b200.runtime import GaweeError
    rng = np.random.default_rng(31)
    for what in ("page", "length"):
        c = Cache(rng, [100, 80], 2, 64, 16, "f32")
        h = c.handle(2)
        n = c.cols * 16
        w = torch.rand((2, 2, n), device="cuda")
        lens, kept = c.lengths(), torch.zeros((2, 2, 40), dtype=torch.int32, device="cuda")
        to = None if in_place else torch.tensor([[0, 0, 0], [0, 0, 0]], dtype=torch.int32, device="cuda")
        if what == "page":
            c.table[0, 6] = 1 << 20
            if to is not None:
                to[:] = c.num_pages
        else:
            lens[0] = n + 1
            if to is not None:
                to[:] = -1
        pages = c.k.clone()
        h.evict(c.k, c.v, w, c.table, lens, 40, 8, kept, torch.zeros_like(w), torch.zeros_like(lens), to_table=to)
        with pytest.raises(GaweeError, match="block table" if what == "page" else "(block table|longer)") as e:
            h.synchronize()
        assert e.value.status == 6
        if not in_place:  # no page to write to
            assert torch.equal(torch.nan_to_num(c.k), torch.nan_to_num(pages))


# --- together -------------------------------------------------------------------

@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_prompts_steps_and_eviction_together(dtype, act):
    """Prompts are appended, steps attend, store and accumulate, the cache is cut
    in place, and steps go on: as a server runs them, nothing in between."""
    rng = np.random.default_rng(40)
    heads, kv, dim, page, batch = 6, 2, 64, 16, 3
    c = Cache(rng, [0] * batch, kv, dim, page, dtype, spare_rows=200)
    h = c.handle(heads, weights=True)
    s = torch.cuda.Stream()
    n = c.cols * page
    prompts = [50, 1, 97]
    k, v = (_normal(rng, (sum(prompts), kv, dim), act).cuda() for _ in range(2))
    seq = torch.tensor([i for i, p in enumerate(prompts) for _ in range(p)], dtype=torch.int32, device="cuda")
    pos = torch.tensor([j for p in prompts for j in range(p)], dtype=torch.int32, device="cuda")
    w = torch.zeros((batch, kv, n), device="cuda")
    torch.cuda.synchronize()
    h.append(c.k, c.v, k, v, c.table, pos, sequences=seq, stream=s)
    at = 0
    for i, p in enumerate(prompts):
        c.rows[i] = [x[at:at + p].transpose(0, 1).cpu().to(T[dtype]) for x in (k, v)]
        at += p
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    budget, recent = 40, 9
    kept = torch.zeros((batch, kv, budget), dtype=torch.int32, device="cuda")
    for step in range(12):
        q = _normal(rng, (batch, heads, dim), act, 2.0).cuda()
        kn, vn = (_normal(rng, (batch, kv, dim), act).cuda() for _ in range(2))
        out = torch.empty_like(q)
        before = w.clone()
        lens += 1
        torch.cuda.synchronize()
        h.attend(c.k, c.v, q, c.table, lens, out, k=kn, v=vn, weights=w, weights_out=w, stream=s)
        h.synchronize(s)
        for i in range(batch):
            for which, x in ((0, kn), (1, vn)):
                c.rows[i][which] = torch.cat([c.rows[i][which], x[i].cpu().to(T[dtype])[:, None]], 1)
        c.lens = lens.cpu().tolist()
        _check_attend(c, q, out, act, dim ** -0.5, None, before, w, before)
        if step % 4 == 3:
            ww = w.cpu().numpy()
            h.evict(c.k, c.v, w, c.table, lens, budget, recent, kept, w, lens, stream=s)
            h.synchronize(s)
            for i, ln in enumerate(c.lens):
                keep = [_kept(ww[i, j], ln, budget, recent) for j in range(kv)]
                for which in (0, 1):
                    c.rows[i][which] = torch.stack([c.rows[i][which][j, keep[j]] for j in range(kv)])
                for pages, which in ((c.k, 0), (c.v, 1)):
                    assert torch.equal(c.get(pages, i, min(ln, budget)), c.rows[i][which])
            c.lens = lens.cpu().tolist()
            assert max(c.lens) <= budget


# --- in a graph ------------------------------------------------------------------

@pytest.mark.parametrize("graph_mode", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("kv_heads,page_size", [(2, 16), (4, 7)])
def test_decode_graph_follows_the_concatenating_step_for_every_length(kv_heads, page_size, graph_mode):
    """One context of llama_decode_paged against the oracle's run of llama_decode
    (the same weights, the cache concatenated), one graph per length."""
    import oracle
    from gawee_b200 import synth
    from gawee_b200.runtime import Model
    from tests.helpers import compare
    batch, layers, heads, dim, start = 2, 2, 4, 128, 3
    kw = dict(batch=batch, dim=dim, layers=layers, heads=heads, kv_heads=kv_heads, ffn=128, vocab=300)
    hd, cols = dim // heads, 4
    g = synth.llama_decode_paged(page_size=page_size, max_pages=cols, num_pages=batch * cols + 1, **kw)
    args = g.make_args()
    rng = np.random.default_rng(50)
    perm = rng.permutation(batch * cols + 1).astype(np.int32)[:batch * cols].reshape(batch, cols)
    past = [rng.standard_normal((batch, kv_heads, start, hd), dtype=np.float32) for _ in range(2 * layers)]
    args[2] = perm
    for i, p in enumerate(past):  # rows 0 .. start - 1 of every layer
        for b in range(batch):
            for r in range(start):
                args[4 + i][perm[b, r // page_size], :, r % page_size] = p[b, :, r]
    m = Model(g.mlir, graph_mode=graph_mode)
    try:
        m.set_args(args)
        for step in range(20):
            n = start + step  # rows cached before this step
            ids = rng.integers(0, 300, (batch, 1), dtype=np.int64)
            pid = np.full((batch, 1), n, np.int64)
            m.set_arg(0, ids)
            m.set_arg(1, pid)
            m.set_arg(3, np.full((batch,), n + 1, np.int32))
            m.forward()
            got = m.output(0)
            m.synchronize()
            ref = synth.llama_decode(past=n, **kw)
            ra = ref.make_args()
            weights = [a for a, s in zip(ra, ref.args) if s.kind == "weight"]
            assert all(np.array_equal(a, b) for a, b in
                       zip(weights, [a for a, s in zip(args, g.args) if s.kind == "weight"]))
            want = oracle.run(ref.mlir, [ids, np.ones((batch, n + 1), np.int64), pid] + past + weights)
            past = list(want[1:])
            compare(got, want[0], atol=5e-4, rtol=1e-4, what=f"logits of step {step}")
    finally:
        m.close()


def test_decode_graph_of_the_15m_shapes_runs_with_the_library_calls_on_its_pages():
    """A prompt appended by gawee_kv_append into the context's own pages, then a step of the graph."""
    from gawee_b200 import runtime, synth
    from gawee_b200.paged_kv import _APPEND, PagedKV
    from gawee_b200.runtime import Model
    g = synth.llama_decode_paged(batch=1, layers=2, vocab=1000, page_size=16, max_pages=4)
    args = g.make_args()
    prompt = 37
    rng = np.random.default_rng(51)
    rows = [torch.from_numpy(rng.standard_normal((prompt, 6, 48), dtype=np.float32)).cuda() for _ in range(4)]
    args[3][:] = prompt + 1
    args[1][:] = prompt
    plain = [a.copy() for a in args]
    for i, r in enumerate(rows):
        for j in range(prompt):
            plain[4 + i][args[2][0, j // 16], :, j % 16] = r[j].cpu().numpy()
    a, b = Model(g.mlir), Model(g.mlir)
    try:
        a.set_args(args)
        kv = PagedKV("f32", 6, 6, 48, 16, 4, max_batch=1, max_pages=4)
        table = torch.from_numpy(args[2]).cuda()
        pos = torch.arange(prompt, dtype=torch.int32, device="cuda")
        seq = torch.zeros(prompt, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        for layer in range(2):
            packed = _APPEND.pack(a.arg_ptr(4 + 2 * layer), a.arg_ptr(5 + 2 * layer), rows[2 * layer].data_ptr(),
                                  rows[2 * layer + 1].data_ptr(), 0, 288, 288, prompt, seq.data_ptr(), pos.data_ptr(),
                                  table.data_ptr(), 4, 4, 1)
            assert runtime.load_library().gawee_kv_append(kv._h, packed, None) == 0
        kv.synchronize()
        a.forward()
        got = a.output(0)
        want = b.run(plain)[0]
        assert np.array_equal(got, want)
    finally:
        a.close()
        b.close()


# --- larger batches and what the division of the work does with them ------------------

@pytest.mark.parametrize("types", TYPES[:3], ids=lambda t: f"{t[0]}-{t[1]}")
def test_attend_many_sequences(types):
    """More sequences than a block has threads, of all lengths, with rows of none between them."""
    rng = np.random.default_rng(60)
    lens = [int(x) for x in rng.choice([-1, 0, 1, 2, 3, 15, 16, 17, 40, 64, 65, 130], 700)]
    lens[0] = lens[1] = lens[-1] = -1
    c = Cache(rng, lens, 2, 32, 16, types[0])
    _run(c, 6, types[1], with_weights=True, new=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_one_long_sequence_among_short_ones(dtype):
    c = Cache(np.random.default_rng(61), [1, 3, 9000, 2, -1, 0, 5, 130], 2, 64, 16, dtype)
    _run(c, 8, dtype, new=True, with_weights=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["all", "front", "back", "all_but_one"])
def test_attend_masks_that_empty_whole_parts(dtype, kind):
    """A mask that leaves some or all of the blocks that share a sequence without a row."""
    c = Cache(np.random.default_rng(62), [6000, 50], 1, 64, 32, dtype)
    mask = np.zeros((2, c.cols * c.page), np.float32)
    mask[0, {"all": slice(None), "front": slice(0, 5900), "back": slice(70, None), "all_but_one": slice(None)}[kind]] = -np.inf
    if kind == "all_but_one":
        mask[0, 4321] = 0
    _run(c, 4, dtype, mask=torch.from_numpy(mask).cuda(), with_weights=True)


@pytest.mark.parametrize("in_place", [False, True], ids=["copied", "in_place"])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd", "rising"])
def test_evict_by_several_blocks_a_head(kind, in_place):
    _evict([9000, 4097, 5, 8999], 2, 8, 64, "f32", 4000, 700, kind, in_place, alias=in_place)
    _evict([9000, 4500], 1, 8, 64, "bf16", 300, 300, kind, in_place)
    _evict([5000], 1, 8, 7, "f16", 4999, 0, kind, in_place, alias=True)


def test_evict_many_long_sequences():
    _evict([4200 + 7 * i for i in range(60)], 1, 8, 64, "bf16", 1000, 100, "ties", True, alias=True)


def test_evict_many_short_sequences():
    _evict([int(x) for x in np.random.default_rng(63).integers(-1, 90, 300)], 2, 8, 16, "f32", 30, 7, "ties", False)


def test_append_many_tokens_of_many_sequences():
    rng = np.random.default_rng(64)
    c = Cache(rng, [0] * 90, 2, 16, 16, "bf16", spare_rows=70)
    new = [(b, p) for b in range(90) for p in range(int(rng.integers(0, 70)))]
    k, v = (_normal(rng, (len(new), 2, 16), "f32").cuda() for _ in range(2))
    seq, pos = (torch.tensor([x[i] for x in new], dtype=torch.int32, device="cuda") for i in (0, 1))
    h = c.handle(2)
    h.append(c.k, c.v, k, v, c.table, pos, sequences=seq)
    h.synchronize()
    at = 0
    for b in range(90):
        n = sum(1 for x in new if x[0] == b)
        for pages, x in ((c.k, k), (c.v, v)):
            assert torch.equal(c.get(pages, b, n), x[at:at + n].transpose(0, 1).to(torch.bfloat16).cpu())
        at += n


def test_calls_leave_the_current_device_and_no_error_behind():
    c = Cache(np.random.default_rng(65), [20], 1, 64, 16, "f32")
    before = torch.cuda.current_device()
    _run(c, 2, "f32")
    assert torch.cuda.current_device() == before
    torch.cuda.synchronize()


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")], ids=lambda t: f"{t[0]}-{t[1]}")
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_new_rows_of_any_alignment_masked_and_on_bad_pages(types, offset):
    """New rows that start on a 16-byte boundary or do not; one that the mask
    takes out (stored all the same), one whose page is bad (not stored)."""
    from gawee_b200.runtime import GaweeError
    rng = np.random.default_rng(70)
    c = Cache(rng, [17, 64, 65, 1, 130], 2, 64, 16, types[0])
    flat = [_normal(rng, (offset + 5 * 136,), types[1]).cuda() for _ in range(2)]
    k, v = (f.as_strided((5, 2, 64), (136, 64, 1), offset) for f in flat)
    q = _normal(rng, (5, 8, 64), types[1]).cuda()
    mask = torch.zeros((5, c.cols * 16), device="cuda")
    mask[1, 63] = -float("inf")
    c.table[4, 8] = c.num_pages + 5
    before = [c.k.clone(), c.v.clone()]
    h = c.handle(8)
    out = h.attend(c.k, c.v, q, c.table, c.lengths(), torch.empty_like(q), k=k, v=v, mask=mask)
    with pytest.raises(GaweeError, match="block table"):
        h.synchronize()
    for i in range(4):
        n = c.lens[i]
        for which, x in ((0, k), (1, v)):
            c.rows[i][which][:, n - 1] = x[i].cpu().to(T[types[0]])
            before[which][int(c.table_np[i, (n - 1) // 16]), :, (n - 1) % 16] = x[i].to(T[types[0]])
    for got, want in zip((c.k, c.v), before):
        assert torch.equal(torch.nan_to_num(got.float(), nan=9.0), torch.nan_to_num(want.float(), nan=9.0))
    c.lens[4] = 128  # its other rows are attended as they are
    _check_attend(c, q, out, types[1], 0.125, mask)


def test_captured_append_step_and_eviction():
    """append, attend with weights and evict in place in one graph, replayed on
    new inputs: as many times as the same calls made one by one."""
    rng = np.random.default_rng(80)
    caches = [Cache(np.random.default_rng(81), [60, 33, 1], 2, 64, 16, "bf16", spare_rows=80) for _ in range(2)]
    state = []
    for c in caches:
        n = c.cols * c.page
        state.append(dict(h=c.handle(8, weights=True), w=torch.zeros((3, 2, n), device="cuda"), lens=c.lengths(),
                          kept=torch.zeros((3, 2, 40), dtype=torch.int32, device="cuda"),
                          q=torch.zeros((3, 8, 64), dtype=torch.bfloat16, device="cuda"),
                          kv=[torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(4)],
                          out=torch.zeros((3, 8, 64), dtype=torch.bfloat16, device="cuda")))

    def step(c, s, stream):
        s["h"].append(c.k, c.v, s["kv"][0], s["kv"][1], c.table, s["lens"], stream=stream)  # one row more ..
        s["lens"] += 2                                                                     # .. and the step's own
        s["h"].attend(c.k, c.v, s["q"], c.table, s["lens"], s["out"], k=s["kv"][2], v=s["kv"][3], weights=s["w"],
                      weights_out=s["w"], stream=stream)
        s["h"].evict(c.k, c.v, s["w"], c.table, s["lens"], 40, 8, s["kept"], s["w"], s["lens"], stream=stream)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(caches[0], state[0], torch.cuda.current_stream())
    for _ in range(6):
        new = [_normal(rng, t.shape, "bf16") for t in [state[0]["q"]] + state[0]["kv"]]
        for s in state:
            for t, x in zip([s["q"]] + s["kv"], new):
                t.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
            step(caches[1], state[1], stream)
        for s in state:
            s["h"].synchronize(stream)
        for name in ("out", "w", "lens", "kept"):
            assert torch.equal(state[0][name], state[1][name]), name
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
            assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))
    assert state[0]["lens"].tolist() == [40, 40, 13]


def test_two_handles_at_the_same_time():
    """Calls that overlap, on two streams with a handle each, as many as the caller likes."""
    cs = [Cache(np.random.default_rng(82 + i), [900, 5, 2000][::1 - 2 * i], 2, 64, 16, ("f32", "bf16")[i]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cs]
    handles = [c.handle(8, weights=True) for c in cs]
    qs = [_normal(np.random.default_rng(1), (3, 8, 64), c.dtype).cuda() for c in cs]
    lens = [c.lengths() for c in cs]
    ws = [torch.zeros((3, 2, c.cols * c.page), device="cuda") for c in cs]
    outs = [[torch.empty_like(q) for _ in range(15)] for q in qs]
    wos = [[torch.zeros_like(w) for _ in range(15)] for w in ws]
    torch.cuda.synchronize()
    for r in range(15):
        for i, c in enumerate(cs):
            handles[i].attend(c.k, c.v, qs[i], c.table, lens[i], outs[i][r], weights=ws[i], weights_out=wos[i][r],
                              stream=streams[i])
    for i, c in enumerate(cs):
        handles[i].synchronize(streams[i])
        for r in range(15):
            assert torch.equal(outs[i][r], outs[i][0]) and torch.equal(wos[i][r], wos[i][0])
        _check_attend(c, qs[i], outs[i][0], c.dtype, 0.125, None, ws[i], wos[i][0], ws[i])
