"""Paged key/value cache without a GPU: what the calls refuse, and where a row lies in the pages.

A handle made for device -1 checks the arguments of its calls and then says
that it has no device, so that every refusal is reached here.
"""
import os
import subprocess

import pytest
import torch

from gawee_b200 import build, runtime
from gawee_b200.paged_kv import PagedKV
from gawee_b200.runtime import GaweeError

INVALID, CUDA = 1, 4
B, H, KV, D, PAGE, PAGES, COLS = 3, 6, 2, 16, 4, 20, 5


def _handle(**kw):
    args = dict(dtype="f32", heads=H, kv_heads=KV, head_dim=D, page_size=PAGE, num_pages=PAGES, max_batch=4,
                max_pages=8, weights=True, device=-1)
    args.update(kw)
    return PagedKV(**args)


def _refused(call, status=INVALID, match=None):
    with pytest.raises(GaweeError, match=match) as e:
        call()
    assert e.value.status == status


@pytest.mark.parametrize("bad", [
    dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(head_dim=12), dict(head_dim=0), dict(head_dim=264),
    dict(page_size=0), dict(page_size=65537), dict(num_pages=0), dict(num_pages=1 << 31), dict(page_stride=1),
    dict(page_stride=KV * PAGE * D + 1), dict(max_batch=0), dict(max_batch=65536), dict(max_pages=0),
    dict(max_pages=1 << 29), dict(page_stride=1 << 61), dict(heads=-6, kv_heads=-2), dict(heads=(1 << 32) + H),
])
def test_create_refuses(bad):
    try:
        kv = _handle(**bad)
    except GaweeError as e:
        assert e.status == INVALID
    else:
        kv.close()
        raise AssertionError("not refused")


def test_create_refuses_type_and_device():
    with pytest.raises(ValueError):
        _handle(dtype="f64")
    _refused(lambda: _handle(device=-2), INVALID if torch.cuda.is_available() else CUDA)


def _attend_args(**kw):
    a = dict(k_pages=torch.zeros(PAGES, KV, PAGE, D), v_pages=torch.zeros(PAGES, KV, PAGE, D), q=torch.zeros(B, H, D),
             block_table=torch.zeros(B, COLS, dtype=torch.int32), lengths=torch.ones(B, dtype=torch.int32),
             out=torch.zeros(B, H, D))
    a.update(kw)
    return a


N = COLS * PAGE
GOOD = [
    {},
    dict(mask=torch.zeros(B, N)), dict(mask=torch.zeros(1, N)), dict(mask=torch.zeros(B, N + 3)[:, :N]),
    dict(k=torch.zeros(B, KV, D), v=torch.zeros(B, KV, D)),
    dict(q=torch.zeros(B, H + 4, D)[:, :H], out=torch.zeros(2 * B, H, D)[::2]),
    dict(weights_out=torch.zeros(B, KV, N)), dict(weights_out=torch.zeros(B, KV, N), weights=torch.zeros(B, KV, N)),
    dict(q=torch.zeros(B, H, D, dtype=torch.bfloat16), out=torch.zeros(B, H, D, dtype=torch.bfloat16)),
    dict(block_table=torch.zeros(B, 9, dtype=torch.int32)[:, :COLS]),
    dict(scale=0.0), dict(scale=-1.0),
]


@pytest.mark.parametrize("kw", GOOD, ids=range(len(GOOD)))
def test_attend_accepts(kw):
    kv = _handle()
    _refused(lambda: kv.attend(**_attend_args(**kw)), CUDA, "no device")


def _unaligned_pages():
    return torch.zeros(PAGES * KV * PAGE * D + 4)[1:1 + PAGES * KV * PAGE * D].view(PAGES, KV, PAGE, D)


BAD = [
    dict(k_pages=torch.zeros(PAGES, KV, PAGE + 1, D)), dict(k_pages=torch.zeros(PAGES, KV, PAGE, D, dtype=torch.float16)),
    dict(k_pages=torch.zeros(PAGES, PAGE, KV, D).transpose(1, 2)), dict(k_pages=_unaligned_pages()),
    dict(k_pages=torch.zeros(PAGES * 2, KV, PAGE, D)[::2]),
    dict(q=torch.zeros(B, H, D + 8)), dict(q=torch.zeros(B, H + 1, D)), dict(q=torch.zeros(B, H, 2 * D)[:, :, ::2]),
    dict(q=torch.zeros(B, H, D, dtype=torch.float64)), dict(q=torch.zeros(B, H, D, dtype=torch.float16)),
    dict(out=torch.zeros(B, H, D, dtype=torch.bfloat16)), dict(out=torch.zeros(1, H, D).expand(B, H, D)),
    dict(block_table=torch.zeros(B + 1, COLS, dtype=torch.int32)), dict(block_table=torch.zeros(B, COLS)),
    dict(block_table=torch.zeros(B, 9, dtype=torch.int32)), dict(block_table=torch.zeros(COLS, B, dtype=torch.int32).t()),
    dict(block_table=torch.zeros(1, COLS, dtype=torch.int32).expand(B, COLS)),
    dict(lengths=torch.ones(B, dtype=torch.int64)), dict(lengths=torch.ones(B + 1, dtype=torch.int32)),
    dict(k=torch.zeros(B, KV, D)), dict(v=torch.zeros(B, KV, D)),
    dict(k=torch.zeros(B, KV, D, dtype=torch.float16), v=torch.zeros(B, KV, D, dtype=torch.float16)),
    dict(k=torch.zeros(B, KV + 1, D), v=torch.zeros(B, KV, D)),
    dict(mask=torch.zeros(B + 1, N)), dict(mask=torch.zeros(B, N, dtype=torch.float16)), dict(mask=torch.zeros(N, B).t()),
    dict(mask=torch.zeros(B, 0)), dict(mask=torch.zeros(B, N, dtype=torch.bool)),
    dict(weights=torch.zeros(B, KV, N)), dict(weights_out=torch.zeros(B, H, N)),
    dict(weights_out=torch.zeros(1, KV, N).expand(B, KV, N)), dict(weights_out=torch.zeros(B, 1, N).expand(B, KV, N)),
    dict(weights_out=torch.zeros(B, KV, N), weights=torch.zeros(B, KV, N + 1)),
    dict(scale=float("nan")), dict(scale=float("inf")),
]


@pytest.mark.parametrize("kw", BAD, ids=range(len(BAD)))
def test_attend_refuses(kw):
    kv = _handle()
    _refused(lambda: kv.attend(**_attend_args(**kw)))


def test_attend_refuses_the_same_pages_twice_a_large_batch_and_weights_of_a_handle_without():
    kv = _handle()
    p = torch.zeros(PAGES, KV, PAGE, D)
    _refused(lambda: kv.attend(**_attend_args(k_pages=p, v_pages=p)))
    _refused(lambda: _handle(max_batch=2).attend(**_attend_args()), match="batch 3")
    _refused(lambda: _handle(weights=False).attend(**_attend_args(weights_out=torch.zeros(B, KV, N))), match="without")
    w = torch.zeros(B * KV * N + N)
    _refused(lambda: kv.attend(**_attend_args(weights=w[:B * KV * N].view(B, KV, N),
                                              weights_out=w.as_strided((B, KV, N - 1), (KV * N, N - 1, 1)))))


def test_empty_batches_are_accepted():
    kv = _handle()
    kv.attend(**_attend_args(q=torch.zeros(0, H, D), out=torch.zeros(0, H, D), lengths=torch.zeros(0, dtype=torch.int32),
                             block_table=torch.zeros(0, COLS, dtype=torch.int32).new_zeros(1, COLS)[:0]))
    t = torch.zeros(B, COLS, dtype=torch.int32)
    pages = [torch.zeros(PAGES, KV, PAGE, D) for _ in range(2)]
    kv.append(*pages, torch.zeros(0, KV, D), torch.zeros(0, KV, D), t, torch.zeros(0, dtype=torch.int32))


def _append_args(**kw):
    a = dict(k_pages=torch.zeros(PAGES, KV, PAGE, D), v_pages=torch.zeros(PAGES, KV, PAGE, D), k=torch.zeros(7, KV, D),
             v=torch.zeros(7, KV, D), block_table=torch.zeros(B, COLS, dtype=torch.int32),
             positions=torch.zeros(7, dtype=torch.int32), sequences=torch.zeros(7, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(sequences=None), dict(positions=torch.zeros(6, dtype=torch.int32)), dict(positions=torch.zeros(7)),
    dict(sequences=torch.zeros(8, dtype=torch.int32)), dict(k=torch.zeros(6, KV, D)),
    dict(v=torch.zeros(7, KV, D, dtype=torch.float16)), dict(k=torch.zeros(1, KV, D).expand(7, KV, D)),
    dict(k=torch.zeros(7, D, KV).transpose(1, 2)), dict(k=torch.zeros(7, KV, D, dtype=torch.int32)),
    dict(block_table=torch.zeros(5, COLS, dtype=torch.int32)), dict(positions=torch.zeros(14, dtype=torch.int32)[::2]),
])
def test_append_refuses(kw):
    kv = _handle()
    _refused(lambda: kv.append(**_append_args()), CUDA, "no device")
    _refused(lambda: kv.append(**_append_args(**kw)))


def _evict_args(**kw):
    a = dict(k_pages=torch.zeros(PAGES, KV, PAGE, D), v_pages=torch.zeros(PAGES, KV, PAGE, D),
             weights=torch.zeros(B, KV, N), block_table=torch.zeros(B, COLS, dtype=torch.int32),
             lengths=torch.ones(B, dtype=torch.int32), budget=6, recent=2, kept=torch.zeros(B, KV, 6, dtype=torch.int32),
             weights_out=torch.zeros(B, KV, N), lengths_out=torch.ones(B, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(budget=0, kept=torch.zeros(B, KV, 0, dtype=torch.int32)), dict(recent=-1), dict(recent=7), dict(budget=5),
    dict(kept=torch.zeros(B, KV, 6)), dict(kept=torch.zeros(B, 6, KV, dtype=torch.int32).transpose(1, 2)),
    dict(weights=torch.zeros(B, H, N)), dict(weights_out=torch.zeros(B, KV, N + 1)),
    dict(lengths_out=torch.ones(B, dtype=torch.int64)), dict(to_table=torch.zeros(B + 1, COLS, dtype=torch.int32)),
    dict(to_table=torch.zeros(B, 9, dtype=torch.int32)), dict(weights_out=torch.zeros(1, KV, N).expand(B, KV, N)),
])
def test_evict_refuses(kw):
    kv = _handle()
    _refused(lambda: kv.evict(**_evict_args()), CUDA, "no device")
    _refused(lambda: kv.evict(**_evict_args(**kw)))


def test_evict_refuses_to_table_that_is_the_table():
    t = torch.zeros(B, COLS, dtype=torch.int32)
    _refused(lambda: _handle().evict(**_evict_args(block_table=t, to_table=t)), match="in place")


def test_null_handles_and_arguments_are_refused():
    lib = runtime.load_library()
    for f in (lib.gawee_kv_append, lib.gawee_kv_attend, lib.gawee_kv_evict):
        assert f(None, None, None) == INVALID
    assert lib.gawee_kv_synchronize(None, None) == INVALID
    assert lib.gawee_kv_create(None, 0, None) == INVALID
    lib.gawee_kv_destroy(None)
    _refused(lambda: _handle().synchronize(), CUDA, "no device")


def test_rows_of_pages_and_bad_pages(tmp_path):
    """page_of and row_offset, the kernels' own index arithmetic, compiled for the host."""
    src = tmp_path / "t.cpp"
    src.write_text("""
#include <cassert>
#include "paged_index.h"
using namespace gawee::kern;
int main() {
  const int32_t table[] = {4, 0, -1, 5, 2147483647, -2147483647 - 1, 3};
  PageGeom g{1000, 5, 3, 7, 16};
  assert(page_of(table, 7, 0, g) == 4 && page_of(table, 7, 6, g) == 4 && page_of(table, 7, 7, g) == 0);
  assert(page_of(table, 7, 13, g) == 0 && page_of(table, 7, 14, g) == -1);  // entry -1
  assert(page_of(table, 7, 21, g) == -1);                                   // entry 5 of 5 pages
  assert(page_of(table, 7, 28, g) == -1 && page_of(table, 7, 35, g) == -1);
  assert(page_of(table, 7, 48, g) == 3 && page_of(table, 7, 49, g) == -1);  // behind the last column
  assert(page_of(table, 7, -1, g) == -1 && page_of(table, 7, 1ll << 40, g) == -1);
  assert(row_offset(4, 2, 6, g) == 4000 + (2 * 7 + 6) * 16);
  PageGeom big{1 << 20, 1 << 20, 8, 128, 128};
  assert(row_offset((1 << 20) - 1, 7, 127, big) == ((1ll << 20) - 1) * (1 << 20) + (7 * 128 + 127) * 128);
}
""")
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(build.CSRC, "kernels"), str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    from gawee_b200 import paged_kv
    src = tmp_path / "s.cpp"
    src.write_text("""
#include <cstdio>
#include "gawee_cuda.h"
int main() {
  printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(gawee_kv_desc), sizeof(gawee_kv_append_args), sizeof(gawee_kv_attend_args),
         sizeof(gawee_kv_evict_args), offsetof(gawee_kv_attend_args, weights_cols), offsetof(gawee_kv_append_args, batch),
         offsetof(gawee_kv_evict_args, kept));
}
""")
    exe = tmp_path / "s"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(build.ROOT, "include"), "-include", "cstddef", str(src), "-o",
                    str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    structs = [paged_kv._DESC, paged_kv._APPEND, paged_kv._ATTEND, paged_kv._EVICT]
    assert [(-(-s.size // 8)) * 8 for s in structs] == got[:4]
    assert got[4:] == [paged_kv._ATTEND.size - 8, paged_kv._APPEND.size - 4, paged_kv._EVICT.size - 8]


def _graph(**kw):
    from gawee_b200 import synth
    return synth.llama_decode_paged(batch=2, layers=2, heads=4, kv_heads=2, dim=128, ffn=128, vocab=64, **kw).mlir


def test_decode_graph_plans_and_merges_its_projections():
    plan = runtime.plan_text(_graph()).split()
    assert plan.count("paged_attention") == 2 and plan.count("matmul3") == 2


def _op_graph(use_pages_again=False, twice=False, computed_pages=False, **kw):
    """One paged_attention op over inputs of the given shapes."""
    from gawee_b200.synth import GraphBuilder
    s = dict(q=(B, H, D), k=(B, KV, D), v=(B, KV, D), k_pages=(PAGES, KV, PAGE, D), v_pages=(PAGES, KV, PAGE, D),
             table=(B, COLS), lengths=(B,), table_type="i32", lengths_type="i32", pages_type="f32")
    s.update(kw)

    def make(g):
        def x(name, dtype="f32"):
            return g.input(dtype, s[name], lambda: None)
        q, k, v, kp, vp = x("q"), x("k"), x("v"), x("k_pages", s["pages_type"]), x("v_pages", s["pages_type"])
        table, lengths = x("table", s["table_type"]), x("lengths", s["lengths_type"])
        pages = g.relu(kp) if computed_pages else kp
        out = [g.paged_attention(q, k, v, pages, kp if twice else vp, table, lengths, 0.5)]
        return out + ([g.relu(vp)] if use_pages_again else [])
    g = GraphBuilder("synthetic:test", 0)
    return g.finish(make(g))


def test_graph_op_plans():
    assert "paged_attention" in runtime.plan_text(_op_graph())
    assert "paged_attention" in runtime.plan_text(_op_graph(q=(B, 7 * KV, D)))


@pytest.mark.parametrize("kw", [
    dict(q=(B, 5, D)), dict(q=(B + 1, H, D)), dict(q=(B, H, D + 8)), dict(q=(B * H, D)), dict(k=(B, KV + 1, D)),
    dict(v=(B, KV, D, 1)), dict(k=(B, 2 * KV, D), v=(B, 2 * KV, D)), dict(table=(B + 1, COLS)), dict(table=(COLS,)),
    dict(table_type="i64"), dict(lengths=(B + 1,)), dict(lengths=(B, 1)), dict(lengths_type="i64"),
    dict(v_pages=(PAGES + 1, KV, PAGE, D)), dict(k_pages=(PAGES, PAGE, KV, D), v_pages=(PAGES, PAGE, KV, D)),
    dict(q=(B, H, 12), k=(B, KV, 12), v=(B, KV, 12), k_pages=(PAGES, KV, PAGE, 12), v_pages=(PAGES, KV, PAGE, 12)),
    dict(q=(B, H, 264), k=(B, KV, 264), v=(B, KV, 264), k_pages=(PAGES, KV, PAGE, 264), v_pages=(PAGES, KV, PAGE, 264)),
    dict(pages_type="f64"), dict(use_pages_again=True), dict(twice=True), dict(computed_pages=True),
])
def test_graph_op_refuses(kw):
    with pytest.raises(GaweeError, match="paged_attention"):
        runtime.plan_text(_op_graph(**kw))
