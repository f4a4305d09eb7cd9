"""A paged decode graph through the calls that stage every argument from host memory."""
import ctypes

import numpy as np
import pytest

from gawee_b200 import synth
from gawee_b200.runtime import GaweeError, Model
from tests.test_gpu_boundary import _result_array, describe, memref_type

pytestmark = pytest.mark.gpu

STEPS = 5


def _graph():
    return synth.llama_decode_paged(batch=2, layers=2, heads=4, kv_heads=2, dim=128, ffn=128, vocab=64, page_size=2,
                                    max_pages=4, num_pages=9)


def _set_step(args, step):
    rng = np.random.default_rng(step)
    args[0][:] = rng.integers(0, 64, args[0].shape)
    args[1][:] = step
    args[3][:] = step + 1


def _stepped(g):
    """Logits of each step, and the pages at the end, of a context that keeps its pages."""
    args = g.make_args()
    m = Model(g.mlir)
    try:
        assert m.in_place_args == [4, 5, 6, 7]
        m.set_args(args)
        got = []
        for step in range(STEPS):
            _set_step(args, step)
            for i in (0, 1, 3):
                m.set_arg(i, args[i])
            m.forward()
            got.append(m.output(0))
        return got, [m.arg(i) for i in m.in_place_args]
    finally:
        m.close()


@pytest.mark.parametrize("how", ["run", "ciface", "embedded"])
def test_a_decode_loop_that_stages_every_argument_keeps_its_rows(cuda_lib, how):
    g = _graph()
    want, pages = _stepped(g)
    args = g.make_args()
    libc = ctypes.CDLL(None)
    libc.free.argtypes = [ctypes.c_void_p]
    text = ctypes.create_string_buffer(g.mlir.encode())  # one address: the context cache key
    m = Model(g.mlir) if how != "embedded" else None
    # the first pages lie behind a descriptor with an offset
    padded = np.zeros(5 + args[4].size, np.float32)
    args[4] = padded[5:].reshape(args[4].shape)
    descs = [describe(a, 5 if i == 4 else 0) for i, a in enumerate(args)]
    ptrs = (ctypes.c_void_p * len(descs))(*[ctypes.addressof(d) for d in descs])
    try:
        for step in range(STEPS):
            _set_step(args, step)
            if how == "run":
                got = m.run(args)[0]
            else:
                res = memref_type(3)()
                st = (cuda_lib.gawee_ciface_forward(m._h, ctypes.addressof(res), ptrs, len(descs)) if how == "ciface" else
                      cuda_lib.gawee_embedded_forward(text, 0, ctypes.addressof(res), ptrs, len(descs)))
                assert st == 0
                got = _result_array(res, want[0].shape, np.float32)
                libc.free(res.allocated)
            assert np.array_equal(got, want[step]), f"step {step}"
        for a, b in zip(args[4:8], pages):
            assert np.array_equal(a, b) and a.any()
        assert not padded[:5].any()
    finally:
        if m is not None:
            m.close()


def test_run_refuses_pages_that_it_cannot_write_and_other_arguments_are_not_read_back():
    g = _graph()
    args = g.make_args()
    m = Model(g.mlir)
    try:
        frozen = args[5].copy()
        frozen.flags.writeable = False
        for bad in (frozen, np.asfortranarray(args[5]), args[5].tolist()):
            with pytest.raises(GaweeError, match="argument 5 is written") as e:
                m.run(args[:5] + [bad] + args[6:])
            assert e.value.status == 1
        m.run(args)
        lib, h = m._lib, m._h
        assert [lib.gawee_arg_in_place(h, i) for i in (-1, 0, 4, 7, 8, len(args))] == [-1, 0, 1, 1, 0, -1]
        assert lib.gawee_arg_in_place(None, 4) == -1
        out = np.empty_like(args[4])
        for call in (lambda: m.arg(0), lambda: m.arg(len(args) - 1), lambda: m.arg(4, out=out[:1]),
                     lambda: m.arg(4, out=np.asfortranarray(out)), lambda: m.arg(4, out=out.astype(np.float64))):
            with pytest.raises(GaweeError) as e:
                call()
            assert e.value.status == 1
        assert lib.gawee_get_arg(h, 4, None, out.nbytes, None) == 1 and lib.gawee_get_arg(None, 4, out.ctypes.data, out.nbytes, None) == 1
        assert lib.gawee_get_arg(h, len(args), out.ctypes.data, out.nbytes, None) == 1
    finally:
        m.close()
