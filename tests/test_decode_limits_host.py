"""What the decoding-step operators promise beside their results, without a GPU."""
import ctypes as C
import os
import re

import pytest

from test_decode_host import P, cache, decode, lib, refused  # noqa: F401  (decode, lib: fixtures)

torch = pytest.importorskip("torch")
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fbgemm_amd", "csrc")


def test_results_over_given_tensors_can_be_traced(decode):  # noqa: F811
    x = torch.empty((2, 10), dtype=torch.bfloat16, device="meta")
    assert decode.penalize_logits(x, out=x) is x
    out = torch.empty((2, 20), dtype=torch.bfloat16, device="meta")[:, ::2]
    got = decode.penalize_logits(x, out=out)
    assert got.shape == (2, 10) and got.stride() == out.stride()
    with pytest.raises(RuntimeError):
        decode.penalize_logits(x, out=out[:, :9])


def test_sizes_are_asked_of_the_tensors_device():
    """The workspace's size goes by the current device: every operator makes its tensors' device that one before it calls the library."""
    text = open(os.path.join(CSRC, "torch_op_decode.cpp")).read()
    bodies = re.split(r"\n(?=[a-zA-Z].*\()", text)
    guarded = [b for b in bodies if "OptionalDeviceGuard" in b]
    assert len(guarded) == 4
    for body in guarded:
        calls = [m.start() for m in re.finditer(r"\bfbgemm_amd_\w+\(", body)]
        assert calls and body.index("OptionalDeviceGuard") < min(calls), body[:80]


def test_caches_whose_rows_overlap_are_refused(lib):  # noqa: F811
    def call(c=None, kc=P, vc=C.c_void_p(1 << 20)):
        s = (C.c_int64 * 2)(128, 64)
        return lib.fbgemm_amd_kv_cache_append(C.byref(c or cache()), P, C.c_void_p(8192), 5, 3, s, s, P, kc, vc, None, None)
    for k in range(3):
        for step in (0, 32):
            strides = [2048, 1024, 64]
            strides[k] = step
            refused(lib, call(cache(key_strides=tuple(strides))), "overlap")
            refused(lib, call(cache(value_strides=tuple(strides))), "overlap")
    refused(lib, call(vc=P), "overlap")
    refused(lib, call(cache(row_ty=2, key_strides=(2176, 1088, 64), value_strides=(2176, 1088, 68))), "overlap")


def test_logits_whose_result_overlaps_them_are_refused(lib):  # noqa: F811
    at = lambda elements: C.c_void_p(1 << 20 | 4 * elements)  # noqa: E731
    def call(logits, out, stride=100, ostride=100, rows=2, vocab=100, mask=None, words=4):
        return lib.fbgemm_amd_penalize_logits(logits, 0, rows, vocab, stride, None, 0, None, None, 64, None, None, None, None, None, 0, None, mask, words,
                                              out, ostride, None)
    for change in ({"out": at(1)}, {"out": at(199)}, {"out": at(100)}, {"logits": at(50)}, {"out": at(0), "ostride": 101}, {"out": at(0), "stride": 0},
                   {"out": at(1), "rows": 1, "stride": 0, "ostride": 0}, {"out": at(150), "stride": 250, "ostride": 250, "vocab": 101, "logits": at(50)},
                   {"out": at(950), "ostride": 0}):
        refused(lib, call(**{"logits": at(0), "out": at(0), **change}), "overlap")
    refused(lib, call(at(0), at(0), mask=P, words=3), "mask")


def test_status_blocks_off_their_boundary_are_refused(lib):  # noqa: F811
    s = (C.c_int64 * 2)(128, 64)
    for at in (4097, 4098, 4100):
        st = C.c_void_p(at)
        refused(lib, lib.fbgemm_amd_kv_block_tables(P, P, 32, 3, P, 4, 4, P, 8, P, 16, 5, P, P, P, P, P, st, None), "status")
        refused(lib, lib.fbgemm_amd_kv_cache_append(C.byref(cache()), P, P, 5, 3, s, s, P, P, C.c_void_p(1 << 20), st, None), "status")
