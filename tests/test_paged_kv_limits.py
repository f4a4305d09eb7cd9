"""Paged key/value cache without a GPU: layouts and refusals at the limits of its types."""
import os
import subprocess

from gawee_b200 import build, paged_kv

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
