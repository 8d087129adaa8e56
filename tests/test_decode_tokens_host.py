"""Rotary positions, 4-bit rows, reading back and sampling without a GPU: what the C ABI refuses before it launches anything, shapes, helpers
and the reference's own sanity."""
import ctypes as C
import math

import numpy as np
import pytest

import decode_tokens_reference as R
from test_decode_host import P, cache, decode, lib, refused  # noqa: F401  (decode, lib: fixtures)

torch = pytest.importorskip("torch")
INT4 = 16  # FBGEMM_AMD_CACHE_INT4
FAR = C.c_void_p(1 << 30)


def cache4(**change):
    return cache(**{"row_ty": INT4, "key_strides": (1152, 576, 36), "value_strides": (1152, 576, 36), **change})


def test_append_of_4_bit_rows_refusals(lib):  # noqa: F811
    def call(c=None, ty=5, kc=P, vc=FAR):
        s = (C.c_int64 * 2)(128, 64)
        return lib.fbgemm_amd_kv_cache_append(C.byref(c or cache4()), P, P, ty, 3, s, s, P, kc, vc, None, None)
    for change, word in (({"c": cache4(dim=63)}, "even"), ({"c": cache4(key_strides=(1152, 576, 38))}, "4-byte"), ({"kc": C.c_void_p(4098)}, "4-byte"),
                         ({"c": cache4(key_strides=(1152, 576, 32))}, "overlap"), ({"c": cache4(value_strides=(1152, 32, 36))}, "overlap"),
                         ({"ty": 2}, "FP32, FP16 or BF16"), ({"vc": None}, "null")):
        refused(lib, call(**change), word)
    s = (C.c_int64 * 2)(128, 64)
    refused(lib, lib.fbgemm_amd_kv_cache_append(C.byref(cache4()), P, C.c_void_p(8192), 5, 3, s, s, P, P, P, None, None), "overlap")


def test_attention_over_4_bit_rows_refusals(lib):  # noqa: F811
    def call(c=None, ty=5, kc=P, size=1 << 30):
        return lib.fbgemm_amd_paged_attention(C.byref(c or cache4()), P, ty, 2, 4, 256, 64, kc, P, P, 3, 3, P, 32, 0.1, 0, 0.0, P, P, P, size, None)
    for change, word in (({"ty": 0}, "FP16 or BF16"), ({"size": 100}, "workspace"), ({"kc": C.c_void_p(4098)}, "4-byte"), ({"c": cache4(dim=60)}, "multiple of 8"),
                         ({"c": cache4(dim=264)}, "256"), ({"c": cache4(key_strides=(1152, 576, 38))}, "4-byte"), ({"c": cache4(dim=7)}, "even")):
        refused(lib, call(**change), word)
    assert lib.fbgemm_amd_paged_attention_workspace(C.byref(cache4()), 5, 4, 3) > 0


def test_read_refusals(lib):  # noqa: F811
    def call(c=None, kc=P, tables=P, width=4, offsets=P, bits=32, requests=2, tokens=5, ty=5, key=P, value=P, status=None):
        return lib.fbgemm_amd_kv_cache_read(C.byref(c or cache()), kc, P, tables, 4, width, offsets, None, bits, requests, tokens, ty, key, value, status, None)
    for change, word in (({"ty": 2}, "FP32, FP16 or BF16"), ({"ty": 0}, "type"), ({"bits": 16}, "index_bits"), ({"requests": -1}, "requests"),
                         ({"requests": 2**31 - 1}, "requests"), ({"tokens": -1}, "tokens"), ({"tokens": 1 << 31}, "tokens"), ({"width": -1}, "2^31"),
                         ({"width": 1 << 28}, "2^31"), ({"kc": None}, "null"), ({"tables": None}, "null"), ({"offsets": None}, "null"), ({"key": None}, "null"),
                         ({"value": C.c_void_p(4104)}, "16-byte"), ({"status": C.c_void_p(4100)}, "status"), ({"kc": C.c_void_p(4097)}, "aligned"),
                         ({"c": cache4(), "kc": C.c_void_p(4098)}, "4-byte"), ({"c": cache4(dim=63)}, "even"), ({"c": cache(row_ty=3)}, "cache holds")):
        refused(lib, call(**change), word)
    assert lib.fbgemm_amd_kv_cache_read(None, P, P, P, 4, 4, P, None, 32, 2, 5, 5, P, P, None, None) < 0
    assert call(tokens=0) == 0


def rows(at=1 << 20, out=1 << 25, heads=2, strides=(256, 64), out_strides=None):
    from fbgemm_amd._lib import HeadRows
    two = C.c_int64 * 2
    return HeadRows(in_=at, out=out, in_strides=two(*strides), out_strides=two(*(out_strides or strides)), heads=heads)


def test_rotate_refusals(lib):  # noqa: F811
    def call(query=None, key=None, ty=5, tokens=3, dim=64, positions=P, bits=64, frequencies=P, pairs=32, magnitude=1.0):
        return lib.fbgemm_amd_rotate_positions(C.byref(query or rows()), None if key is None else C.byref(key), ty, tokens, dim, positions, bits, frequencies, pairs,
                                               0, magnitude, 0, None)
    for change, word in (({"ty": 2}, "FP32, FP16 or BF16"), ({"bits": 8}, "index_bits"), ({"tokens": -1}, "tokens"), ({"tokens": 1 << 31}, "tokens"),
                         ({"dim": 0}, "dim"), ({"dim": 1 << 17}, "dim"), ({"pairs": 33}, "pairs"), ({"pairs": -1}, "pairs"), ({"dim": 4096, "pairs": 1025}, "1024"),
                         ({"magnitude": math.inf}, "magnitude"), ({"positions": None}, "null"), ({"frequencies": None}, "null"),
                         ({"query": rows(at=None)}, "null"), ({"query": rows(out=None)}, "null"), ({"query": rows(strides=(-1, 64))}, "strides"),
                         ({"query": rows(heads=-1)}, "heads"), ({"query": rows(heads=1 << 14), "dim": 1 << 15, "pairs": 4}, "2^28"),
                         ({"query": rows(at=(1 << 20) + 1)}, "aligned"), ({"query": rows(out_strides=(256, 60))}, "overlap"),
                         ({"query": rows(out_strides=(100, 64))}, "overlap"),
                         ({"query": rows(out=(1 << 20) + 64)}, "overlap"),                       # its input's elements, not its own
                         ({"query": rows(out=1 << 20, out_strides=(128, 64))}, "overlap"),
                         ({"query": rows(out=1 << 21), "key": rows(at=1 << 21, out=1 << 22)}, "overlap"),  # what is read as keys
                         ({"key": rows(at=1 << 22, out=1 << 25)}, "overlap")):                             # both results in one place
        refused(lib, call(**change), word)
    assert call(tokens=0) == 0 and call(query=rows(heads=0)) == 0
    assert lib.fbgemm_amd_rotate_positions(None, None, 5, 3, 64, P, 64, P, 32, 0, 1.0, 0, None) < 0


def test_sample_refusals(lib):  # noqa: F811
    def call(logits=P, ty=0, rows=2, vocab=100, stride=100, uniform=P, tokens=P, logs=P):
        return lib.fbgemm_amd_sample_tokens(logits, ty, rows, vocab, stride, uniform, None, None, None, None, tokens, logs, None)
    for change, word in (({"ty": 2}, "FP32, FP16 or BF16"), ({"rows": -1}, "rows"), ({"rows": (1 << 24) + 1}, "rows"), ({"vocab": 0}, "vocab"),
                         ({"vocab": (1 << 20) + 1}, "vocab"), ({"logits": None}, "null"), ({"uniform": None}, "null"), ({"tokens": None}, "null"),
                         ({"logs": None}, "null"), ({"stride": -1}, "strides")):
        refused(lib, call(**change), word)
    assert call(rows=0) == 0


def test_shapes_of_the_torch_operators(decode):  # noqa: F811
    m = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    q, k = m([3, 8, 64], torch.float16), m([3, 2, 64], torch.float16)
    got = decode.rotate_positions(q, k, m([3], torch.int64), m([32], torch.float64))
    assert [(tuple(x.shape), x.dtype) for x in got] == [((3, 8, 64), torch.float16), ((3, 2, 64), torch.float16)]
    got = decode.rotate_positions(q, k, m([3], torch.int64), m([32], torch.float64), out=(q, k))
    assert got[0] is q and got[1] is k
    with pytest.raises(RuntimeError):
        decode.rotate_positions(q, k, m([3], torch.int64), m([32], torch.float64), out=(k, q))
    c4 = m([4, 2, 16, 36], torch.uint8)
    for dtype, want in ((None, torch.float32), (torch.bfloat16, torch.bfloat16)):
        got = decode.kv_cache_read(c4, c4, m([3, 5], torch.int32), m([4], torch.int32), 7, 64, dtype, row_bits=4)
        assert [(tuple(x.shape), x.dtype) for x in got] == [((7, 2, 64), want)] * 2
    got = decode.kv_cache_read(m([4, 2, 16, 64], torch.float16), m([4, 2, 16, 64], torch.float16), m([3, 5], torch.int32), m([4], torch.int32), 7, 64)
    assert got[1].dtype == torch.float16
    out, lse = decode.paged_attention(q, c4, c4, m([3, 5], torch.int32), m([3], torch.int32), row_bits=4)
    assert out.shape == (3, 8, 64) and lse.shape == (3, 8)
    assert decode.kv_cache_append(k, k, c4, c4, m([3], torch.int64), row_bits=4) is None
    s = decode.sample_tokens(m([3, 1000], torch.bfloat16), m([3], torch.float32))
    assert s.tokens.dtype == torch.int64 and s.log_probabilities.dtype == torch.float32 and s.tokens.shape == s.log_probabilities.shape == (3,)


def test_row_bytes(decode):  # noqa: F811
    assert [decode.kv_row_bytes(d, 4) for d in (2, 8, 10, 64, 128)] == [8, 8, 12, 36, 68]
    for bad in ((64, 2), (7, 4)):
        with pytest.raises(ValueError):
            decode.kv_row_bytes(*bad)


def test_frequencies(decode):  # noqa: F811
    f = decode.rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1 and abs(float(f[16]) - 0.01) < 1e-16
    assert torch.allclose(decode.rotary_frequencies(64, factor=4.0, device="cpu"), f / 4, rtol=1e-15, atol=0)
    g = decode.rotary_frequencies(64, factor=8.0, trained=8192, low=1.0, high=4.0, device="cpu")
    waves = 8192 * f / (2 * math.pi)
    assert torch.equal(g[waves >= 4], f[waves >= 4]) and torch.allclose(g[waves <= 1], f[waves <= 1] / 8, rtol=1e-15, atol=0)
    between = (waves > 1) & (waves < 4)
    assert between.any() and (g[between] < f[between]).all() and (g[between] > f[between] / 8).all() and (g[1:] < g[:-1]).all()
    for bad in ({"dim": 7}, {"dim": 0}, {"dim": 8, "base": 0.0}, {"dim": 8, "factor": -1.0}, {"dim": 8, "trained": 100, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            decode.rotary_frequencies(device="cpu", **bad)


def test_reference_of_rotation_by_hand():
    x = np.array([[[1.0, 0.0, 5.0, 2.0, 0.0]]])
    for inter, want in ((True, [0.0, 2.0, -4.0, 10.0, 0.0]), (False, [-10.0, 0.0, 0.0, 2.0, 0.0])):
        f = [math.pi / 6, math.pi / 6] if inter else [math.pi / 6, 0.0]
        got, _ = R.rotate(x, np.array([3]), f, inter, 2.0)
        assert np.allclose(got, [[want]]) if inter else np.allclose(got, [[[-10.0, 0.0, 2.0, 4.0, 0.0]]])
        back, _ = R.rotate(got, np.array([3]), f, inter, 0.5, inverse=True)
        assert np.allclose(back, x)


def test_reference_of_sampling_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    at = lambda u, t, **k: R.Sampled(x, **k).holds(t, u, np.log(p))  # noqa: E731
    for u, t, p in ((0.0, 0, 0.1), (0.09, 0, 0.1), (0.11, 1, 0.4), (0.49, 1, 0.4), (0.51, 2, 0.2), (0.71, 3, 0.3), (1.0, 3, 0.3)):
        assert at(u, t) and not at(u, (t + 1) % 4)
    p = 4 / 7
    assert at(0.5, 1, top_k=2) and not at(0.5, 2, top_k=2)
    assert at(0.5, 1, top_p=0.65)  # 0.4 and 0.3
    p = 0.4 / 0.9
    assert at(0.3, 1, top_p=0.75) and at(0.3, 1, min_p=0.5)  # 0.4, 0.3 and 0.2
    p = 1.0
    assert at(0.9, 1, temperature=0.0) and at(0.2, 1, min_p=1.0) and at(0.2, 1, top_p=0.0)
    assert R.Sampled(np.array([-np.inf, np.nan])).holds(-1, 0.5, -np.inf)
