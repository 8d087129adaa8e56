"""The decoding-step operators without a GPU: what the C ABI refuses before it launches anything, the shapes the torch
operators report, and the reference that the GPU tests hold them to."""
import ctypes as C
import os

import numpy as np
import pytest

import decode_reference as R

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import build
    if not os.path.exists(build.TORCH_OP_OUT):
        build.build_library()
        build.build_torch_op()
    from fbgemm_amd import decode as d
    return d


@pytest.fixture(scope="module")
def lib(decode):
    import fbgemm_amd
    return fbgemm_amd.lib()


def cache(**change):
    from fbgemm_amd._lib import PagedCache
    values = dict(row_ty=5, block_size=16, heads=2, dim=64, blocks=4, key_strides=(2048, 1024, 64), value_strides=(2048, 1024, 64))
    values.update(change)
    values["key_strides"] = (C.c_int64 * 3)(*values["key_strides"])
    values["value_strides"] = (C.c_int64 * 3)(*values["value_strides"])
    return PagedCache(**values)


def refused(lib, rc, word):
    assert rc < 0
    assert word in lib.fbgemm_amd_last_error().decode(), lib.fbgemm_amd_last_error()


P = C.c_void_p(4096)  # never looked at: the calls are refused first


def test_block_tables_refusals(lib):
    def call(lengths=P, bits=32, requests=3, width=4, stride=4, free_numel=8, block=16, tokens=5, slots=P):
        return lib.fbgemm_amd_kv_block_tables(lengths, P, bits, requests, P, stride, width, P, free_numel, P, block, tokens, slots, P, P, P, P, None, None)
    for change, word in (({"bits": 16}, "index_bits"), ({"requests": -1}, "requests"), ({"block": 0}, "block_size"), ({"block": 1 << 21}, "block_size"),
                         ({"width": -1}, "2^31"), ({"width": 1 << 28}, "2^31"), ({"stride": 3}, "overlap"), ({"free_numel": -1}, "free list"),
                         ({"tokens": -1}, "num_tokens"), ({"tokens": 1 << 31}, "num_tokens"), ({"lengths": None}, "null"), ({"slots": None}, "null")):
        refused(lib, call(**change), word)


def test_append_refusals(lib):
    def call(c=None, ty=5, tokens=3, key=P, strides=(128, 64), kc=P):
        s = (C.c_int64 * 2)(*strides)
        return lib.fbgemm_amd_kv_cache_append(C.byref(c or cache()), key, P, ty, tokens, s, s, P, kc, P, None, None)
    for change, word in (({"ty": 2}, "FP32, FP16 or BF16"), ({"ty": 1}, "type"), ({"tokens": -1}, "tokens"), ({"key": None}, "null"), ({"kc": None}, "null"),
                         ({"strides": (-1, 64)}, "strides"), ({"key": C.c_void_p(4097)}, "aligned"), ({"c": cache(row_ty=3)}, "cache holds"),
                         ({"c": cache(dim=0)}, "dim"), ({"c": cache(heads=0)}, "heads"), ({"c": cache(block_size=0)}, "block_size"),
                         ({"c": cache(blocks=-1)}, "blocks"), ({"c": cache(key_strides=(2048, -1024, 64))}, "strides"),
                         ({"c": cache(row_ty=2, key_strides=(2176, 1088, 67))}, "4-byte"),
                         ({"c": cache(row_ty=2, key_strides=(2176, 1088, 68), value_strides=(2176, 1088, 68)), "kc": C.c_void_p(4098)}, "4-byte")):
        refused(lib, call(**change), word)
    assert lib.fbgemm_amd_kv_cache_append(None, P, P, 5, 1, None, None, P, P, P, None, None) < 0
    assert call(tokens=0) == 0


def test_attention_refusals(lib):
    def call(c=None, ty=5, requests=2, heads=4, stride=256, width=3, bits=32, scale=0.1, window=0, softcap=0.0, query=P, out=P, space=P, size=1 << 30):
        return lib.fbgemm_amd_paged_attention(C.byref(c or cache()), query, ty, requests, heads, stride, 64, P, P, P, width, width, P, bits, scale, window,
                                              softcap, out, P, space, size, None)
    for change, word in (({"ty": 0}, "FP16 or BF16"), ({"ty": 1}, "type"), ({"requests": -1}, "requests"), ({"heads": 3}, "multiple"), ({"heads": 0}, "multiple"),
                         ({"width": -1}, "table_width"), ({"bits": 8}, "index_bits"), ({"scale": float("inf")}, "scale"), ({"window": -1}, "window"),
                         ({"softcap": -1.0}, "softcap"), ({"softcap": float("nan")}, "softcap"), ({"query": None}, "null"), ({"space": None}, "null"),
                         ({"size": 100}, "workspace"), ({"stride": 260}, "16-byte"), ({"query": C.c_void_p(4104)}, "16-byte"), ({"out": C.c_void_p(4104)}, "16-byte"),
                         ({"c": cache(dim=60)}, "multiple of 8"), ({"c": cache(dim=264)}, "256"), ({"c": cache(row_ty=0)}, "FP16, BF16 or INT8"),
                         ({"c": cache(key_strides=(2048, 1024, 60))}, "16-byte")):
        refused(lib, call(**change), word)
    assert call(requests=0) == 0
    assert lib.fbgemm_amd_paged_attention_workspace(C.byref(cache()), 0, 4, 3) == 0
    assert lib.fbgemm_amd_paged_attention_workspace(C.byref(cache()), 5, 4, 3) > 0
    assert lib.fbgemm_amd_paged_attention_workspace(C.byref(cache()), 5, 3, 3) < 0


def test_logits_refusals(lib):
    def call(ty=0, rows=2, vocab=100, stride=100, tokens=P, n=4, offsets=P, bits=64, ids=None, values=None, biases=0, boff=None, mask=None, words=4, out=P, ostride=100):
        return lib.fbgemm_amd_penalize_logits(P, ty, rows, vocab, stride, tokens, n, offsets, None, bits, None, None, None, ids, values, biases, boff, mask,
                                              words, out, ostride, None)
    for change, word in (({"ty": 2}, "FP32, FP16 or BF16"), ({"rows": -1}, "rows"), ({"vocab": 1 << 31}, "vocab"), ({"bits": 16}, "index_bits"), ({"n": -1}, "lists"),
                         ({"out": None}, "null"), ({"stride": 99}, "overlap"), ({"ostride": 99}, "overlap"), ({"offsets": None}, "offsets"),
                         ({"biases": 3}, "biases"), ({"mask": P, "words": 3}, "mask")):
        refused(lib, call(**change), word)
    assert call(rows=0) == 0 and call(vocab=0) == 0


def test_shapes_of_the_torch_operators(decode):
    m = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    t = decode.kv_block_tables(m([3], torch.int64), m([3], torch.int64), m([3, 5], torch.int32), m([9], torch.int32), m([1], torch.int32), 16, 7)
    assert [(tuple(x.shape), x.dtype) for x in t] == [((7,), torch.int64), ((7,), torch.int64), ((4,), torch.int32), ((3,), torch.int64), ((1,), torch.int32)]
    kv = m([4, 2, 16, 64], torch.float16)
    out, lse = decode.paged_attention(m([3, 8, 64], torch.float16), kv, kv, m([3, 5], torch.int32), m([3], torch.int32))
    assert out.shape == (3, 8, 64) and out.dtype == torch.float16 and lse.shape == (3, 8) and lse.dtype == torch.float32
    assert decode.penalize_logits(m([2, 10], torch.bfloat16)).dtype == torch.bfloat16
    assert decode.kv_cache_append(m([3, 2, 64], torch.float16), m([3, 2, 64], torch.float16), kv, kv, m([3], torch.int64)) is None
    assert [decode.kv_row_bytes(d) for d in (1, 4, 7, 64, 128)] == [8, 8, 12, 68, 132]


def test_reference_of_attention_is_softmax():
    rng = np.random.default_rng(0)
    q, kc, vc = rng.standard_normal((1, 2, 8)), rng.standard_normal((3, 1, 4, 8)), rng.standard_normal((3, 1, 4, 8))
    out, lse, _, _ = R.attention(q, kc, vc, np.array([[2, 0]]), np.array([6]), 0.5, window=5)
    k, v = np.concatenate([kc[2, 0], kc[0, 0]])[1:6], np.concatenate([vc[2, 0], vc[0, 0]])[1:6]
    s = torch.from_numpy(0.5 * q[0] @ k.T)
    assert np.allclose(out[0], torch.softmax(s, -1).numpy() @ v) and np.allclose(lse[0], torch.logsumexp(s, -1).numpy())


def test_reference_of_logits_by_hand():
    x, off = R.logits(np.array([[2.0, -2.0, 1.0, 4.0]]), np.array([1, 0, 0, 1]), np.array([0, 4]), np.array([1]), [2.0], [0.25], [0.5],
                      np.array([2, 2]), np.array([9.0, 1.0]), np.array([0, 2]), np.array([[0b0111]]))
    assert x.tolist() == [[2.0 / 2 - 0.5 - 0.5, -4.0 - 0.25 - 0.5, 2.0, -np.inf]]


def test_reference_of_block_tables_by_hand():
    tables, slots, positions, offsets, total, start, bits = R.block_tables(
        np.array([3, 0, 4]), np.array([2, 0, 1]), np.array([[5, -1], [-1, -1], [6, -1]], np.int32), np.array([9, 8, 7], np.int32), 1, 4, 4)
    assert tables.tolist() == [[5, 8], [-1, -1], [6, 7]] and slots.tolist() == [23, 32, 28, -1] and positions.tolist() == [3, 4, 4, 0]
    assert offsets.tolist() == [0, 2, 2, 3] and total.tolist() == [5, 0, 5] and start == 3 and bits == 4
