"""Paged key/value cache without a GPU: layouts and refusals at the limits of its types."""
import os
import subprocess

import pytest

from gawee_b200 import build, paged_kv, runtime
from tests.test_paged_kv import _attend_args, _evict_args, _handle, _op_graph

STRUCTS = {"gawee_kv_desc": paged_kv._DESC, "gawee_kv_append_args": paged_kv._APPEND,
           "gawee_kv_attend_args": paged_kv._ATTEND, "gawee_kv_evict_args": paged_kv._EVICT}


def test_packed_arguments_are_as_long_as_the_structures(tmp_path):
    """The library copies whole structures: the packed bytes hold their padding too."""
    src = tmp_path / "s.cpp"
    src.write_text('#include <cstdio>\n#include "gawee_cuda.h"\nint main() {\n'
                   + "".join(f'  printf("%zu\\n", sizeof({name}));\n' for name in STRUCTS) + "}\n")
    exe = tmp_path / "s"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(build.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [s.size for s in STRUCTS.values()]


@pytest.mark.parametrize("budget,status", [(0, 1), (-1, 1), (1, 4), ((1 << 31) - (1 << 24) - 1, 4), ((1 << 31) - (1 << 24), 1),
                                           ((1 << 31) - 1, 1)])
def test_evict_refuses_budgets_that_the_kernels_indices_would_pass(budget, status):
    """A handle without a device: 1 is a refused argument, 4 the missing device behind the checks.
    A block of the move goes on by 16 x 148 blocks of up to 1024 rows, in 32 bits."""
    kv = paged_kv.PagedKV("bf16", 2, 1, 8, 16, 64, 4, 8, device=-1)
    some = 1 << 20  # an address that nothing reads
    packed = paged_kv._EVICT.pack(some, 2 * some, some, 64, 64, some, 64, 64, 64, 2, some, 8, 8, 0, 0, 0, some, some, budget,
                                  0, some)
    assert runtime.load_library().gawee_kv_evict(kv._h, packed, None) == status


@pytest.mark.parametrize("old,new", [
    ("scale = 0.5 : f64", "scale = 1.0e39 : f64"), ("scale = 0.5 : f64", "scale = -1.0e400 : f64"),
    ("scale = 0.5 : f64", "scale = true"), ("scale = 0.5 : f64", 'scale = "0.5"'), ("scale = 0.5 : f64", "scale = [0.5]"),
    ("-> tensor<3x6x16xf32>\n    return", "-> tensor<3x6x16xf16>\n    return"),
])
def test_graph_op_refuses_a_scale_that_is_no_finite_number_and_other_results(old, new):
    """gawee_kv_attend refuses such a scale too; taken as it was, it became 0 or infinity."""
    text = _op_graph()
    for scale in ("0.5 : f64", "-2 : i64", "0.0 : f32"):
        assert "paged_attention" in runtime.plan_text(text.replace("0.5 : f64", scale))
    assert text.count(old) == 1
    text = text.replace(old, new)
    with pytest.raises(runtime.GaweeError, match="paged_attention"):
        runtime.plan_text(text.replace("return %0 : tensor<3x6x16xf32>", "return %0 : tensor<3x6x16xf16>")
                          if "f16" in new else text)


def test_the_lane_forms_and_their_launches_go_by_one_rule(tmp_path):
    """Which lane form a head dim takes and how many launches a call makes, compiled for the host."""
    src = tmp_path / "r.cpp"
    src.write_text("""
#include <cassert>
#include "paged_kv.h"
using namespace gawee::kern;
int main() {
  for (int d = 8; d <= 256; d += 8) {
    const int lanes = kv_row_lanes(d), tile = kKvWarps * kv_warp_keys(lanes);
    assert(8 * lanes >= d && (lanes == 4 || 4 * lanes < d));  // eight elements a lane hold a row, half as many lanes do not
    assert(tile == (d <= 32 ? 128 : d <= 64 ? 64 : d <= 128 ? 32 : 16));
    assert(kv_attend_launches_f32(d, 1) == 1 && kv_attend_launches_f32(d, tile) == 1);
    assert(kv_attend_launches_f32(d, tile + 1) == 2 && kv_attend_launches_f32(d, 1ll << 40) == 2);
  }
}
""")
    exe = tmp_path / "r"
    cuda = os.path.join(os.path.dirname(os.path.dirname(build.nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(build.CSRC, "kernels"), "-I", cuda, str(src), "-o", str(exe)],
                   check=True)
    subprocess.run([str(exe)], check=True)


@pytest.mark.parametrize("call,kw", [
    ("attend", dict(scale=1e39)), ("attend", dict(scale=-1e300)), ("attend", dict(scale="0.5")),
    ("attend", dict(scale=1 << 2000)), ("evict", dict(budget=6.0)), ("evict", dict(recent=1.5)),
])
def test_numbers_that_their_c_type_cannot_hold_are_refused_like_other_arguments(call, kw):
    kv = _handle()
    args = (_attend_args if call == "attend" else _evict_args)(**kw)
    with pytest.raises(runtime.GaweeError) as e:
        getattr(kv, call)(**args)
    assert e.value.status == 1 and next(iter(kw)) in str(e.value)
