"""Which layouts of queries, keys and their results ``rotate_positions`` takes: what shares a byte is refused, what does not is not. The same of ``kv_cache_read``. And which
caches ``paged_attention`` reads as runs of bytes."""
import ctypes as C
import itertools
import random

import pytest

from test_decode_host import P, cache, decode, lib, refused  # noqa: F401  (decode, lib: fixtures)

torch = pytest.importorskip("torch")
BASE, ELEMENT = 1 << 24, 2


def rows(at, strides, heads, out=None, out_strides=None):
    """Elements behind BASE; strides (tokens, heads) in elements; a result in place, or behind BASE too."""
    from fbgemm_amd._lib import HeadRows
    two = C.c_int64 * 2
    address = lambda n: BASE + ELEMENT * n  # noqa: E731
    return HeadRows(in_=address(at), out=address(at if out is None else out), in_strides=two(*strides), out_strides=two(*(out_strides or strides)), heads=heads)


def call(lib, tokens, dim, query, key=None):  # noqa: F811
    return lib.fbgemm_amd_rotate_positions(C.byref(query), None if key is None else C.byref(key), 5, tokens, dim, P, 64, P, 0, 0, 1.0, 0, None)


def taken(lib, *args):  # noqa: F811
    """Every check is passed: only the launch fails, without a device."""
    assert call(lib, *args) == -2, lib.fbgemm_amd_last_error()
    assert "launch" in lib.fbgemm_amd_last_error().decode()


without_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses are made up: a device would run the calls that are taken")


@without_gpu
@pytest.mark.parametrize("tokens", [1, 2, 5, 64])
def test_parts_of_one_projection_are_taken(lib, tokens):  # noqa: F811
    H, D = 8, 64
    # [tokens, heads, 3, dim]: a head's query, key and value side by side; the same with a gap behind each token
    for token in (H * 3 * D, H * 3 * D + 40):
        query, key = rows(0, (token, 3 * D), H), rows(D, (token, 3 * D), H)
        taken(lib, tokens, D, query, key)
        # the keys' results where the values were
        taken(lib, tokens, D, query, rows(D, (token, 3 * D), H, out=2 * D))
        # contiguous ones into such a buffer
        far = 1 << 20
        taken(lib, tokens, D, rows(far, (H * D, D), H, 0, (token, 3 * D)), rows(2 * far, (H * D, D), H, D, (token, 3 * D)))
        # fewer key heads: every fourth head has one
        taken(lib, tokens, D, query, rows(D, (token, 12 * D), H // 4))
    # [tokens, heads + 2 * kv_heads, dim], its transpose, and [heads, tokens, 3, dim]
    taken(lib, tokens, D, rows(0, (12 * D, D), H), rows(H * D, (12 * D, D), 2))
    taken(lib, tokens, D, rows(0, (D, tokens * D), H), rows(H * tokens * D, (D, tokens * D), 2))
    taken(lib, tokens, D, rows(0, (3 * D, tokens * 3 * D), H), rows(D, (3 * D, tokens * 3 * D), H))
    # every other token of a buffer, its result in the tokens between
    taken(lib, tokens, D, rows(0, (2 * H * D, D), H, out=H * D))
    # one head
    taken(lib, tokens, D, rows(0, (3 * D, D), 1), rows(D, (3 * D, D), 1))


@pytest.mark.parametrize("tokens", [1, 2, 5, 64])
def test_parts_that_share_an_element_are_refused(lib, tokens):  # noqa: F811
    H, D = 8, 64
    for token in (H * 3 * D, H * 3 * D + 40):
        for at in (0, 1, D - 1, 2 * D + 1, 3 * D - 1, 3 * D, 6 * D + 1):
            refused(lib, call(lib, tokens, D, rows(0, (token, 3 * D), H), rows(at, (token, 3 * D), H)), "overlap")
        for out in (-1, 1, D - 1, 2 * D + 1, 3 * D):
            refused(lib, call(lib, tokens, D, rows(0, (token, 3 * D), H, out)), "overlap")
        refused(lib, call(lib, tokens, D, rows(0, (token, 3 * D), H), rows((H - 1) * 3 * D, (token, 3 * D), 1)), "overlap")
    refused(lib, call(lib, tokens, D, rows(0, (12 * D, D), H), rows(H * D - 1, (12 * D, D), 2)), "overlap")
    refused(lib, call(lib, tokens, D, rows(0, (12 * D, D), H, 0, (3 * D, 3 * D))), "overlap")


def elements(at, strides, tokens, heads, dim):
    return {at + t * strides[0] + h * strides[1] + d for t in range(tokens) for h in range(heads) for d in range(dim)}


def test_whatever_shares_an_element_is_refused(lib):  # noqa: F811
    """Small layouts of any steps against their elements, listed. (Layouts that share none may be refused, where they are laid out differently.)"""
    rng = random.Random(5)
    met = 0
    for _ in range(4000):
        tokens, dim, heads = rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 3, 8]), [rng.choice([1, 2, 3, 4]) for _ in "qk"]
        step = lambda: rng.choice([dim, 2 * dim, 3 * dim, dim + 1, 4 * dim, 12 * dim, 12 * dim + 1, 24 * dim, rng.randint(1, 40)])  # noqa: E731
        strides = [(step(), step()) for _ in range(3)]
        if rng.random() < 0.5:
            strides = strides[:1] * 3
        at = [rng.randint(0, 60) * rng.choice([1, dim]) for _ in range(3)]
        query = rows(at[0], strides[0], heads[0], at[1], strides[1])
        key = rows(at[2], strides[2], heads[1])
        read = [elements(at[0], strides[0], tokens, heads[0], dim), elements(at[2], strides[2], tokens, heads[1], dim)]
        written = [elements(at[1], strides[1], tokens, heads[0], dim), read[1]]
        same = at[0] == at[1] and (tokens == 1 or strides[0][0] == strides[1][0]) and (heads[0] == 1 or strides[0][1] == strides[1][1])
        twice = any(len(w) < tokens * n * dim for w, n in zip(written, heads))
        if twice or (read[0] & written[0] and not same) or read[0] & written[1] or read[1] & written[0] or written[0] & written[1]:
            met += 1
            refused(lib, call(lib, tokens, dim, query, key), "overlap")
    assert met > 1000


@without_gpu
def test_layouts_of_equal_steps_are_decided_exactly(lib):  # noqa: F811
    """Queries and keys in place, in one buffer of the same steps: taken just where they share no element."""
    D = 4
    for tokens, heads, kv_heads, token, head in itertools.product((1, 2, 3), (1, 2, 4), (1, 2), (16, 17, 24, 48), (4, 5, 8, 12)):
        if (heads - 1) * head + D > token:
            continue
        query = elements(0, (token, head), tokens, heads, D)
        for at in range(0, 3 * token + 5):
            key = rows(at, (token, head), kv_heads)
            if query & elements(at, (token, head), tokens, kv_heads, D):
                refused(lib, call(lib, tokens, D, rows(0, (token, head), heads), key), "overlap")
            else:
                taken(lib, tokens, D, rows(0, (token, head), heads), key)


@pytest.mark.parametrize("row_ty,row", [(2, lambda d: d + 4), (16, lambda d: d // 2 + 4)])
def test_rows_without_gaps_are_read_as_runs_however_far_apart_pages_are(lib, row_ty, row):  # noqa: F811
    """The faster form (a tenth of a call over long contexts) asks for nothing but a page's rows behind each other, 16 of them or a multiple."""
    form = lambda **c: lib.fbgemm_amd_paged_attention_form(C.byref(cache(row_ty=row_ty, **c)))  # noqa: E731
    for dim in (64, 128, 256):
        n, runs = row(dim), 1 if (row_ty, dim) == (16, 64) else 2
        page = 2 * 16 * n
        for keys, values in (((page, 16 * n, n),) * 2, ((page, 16 * n, n), (2 * page, 16 * n, n)), ((3 * page, 48 * n, n), (2 * page, 32 * n, n)),
                             ((page + 4, 16 * n, n), (page, 16 * n, n))):
            assert form(dim=dim, key_strides=keys, value_strides=values) == runs
        for keys, values in (((2 * page, 16 * n, n + 4), (page, 16 * n, n)), ((page, 16 * n, n), (2 * page, 16 * n, n + 4)), ((page, n, 2 * n),) * 2):
            assert form(dim=dim, key_strides=keys, value_strides=values) == 1
        assert form(dim=dim, block_size=24, key_strides=(48 * n, 24 * n, n), value_strides=(48 * n, 24 * n, n)) == 0
    n = row(96)
    assert form(dim=96, key_strides=(32 * n, 16 * n, n), value_strides=(32 * n, 16 * n, n)) == 1
    assert lib.fbgemm_amd_paged_attention_form(C.byref(cache())) == 1 and lib.fbgemm_amd_paged_attention_form(C.byref(cache(dim=60))) < 0


def read_call(lib, key, value, key_cache, value_cache, tokens=5, **change):  # noqa: F811
    at = lambda n: C.c_void_p(BASE + n)  # noqa: E731
    return lib.fbgemm_amd_kv_cache_read(C.byref(cache(**change)), at(key_cache), at(value_cache), P, 4, 4, P, None, 32, 2, tokens, 5, at(key), at(value), None, None)


READ = 5 * 2 * 64 * 2  # bytes of a result
HELD = 4 * 2048 * 2    # of a cache
CACHES4 = dict(row_ty=16, key_strides=(1152, 576, 36), value_strides=(2304, 576, 36))
HELD4 = 4 * 1152, 3 * 2304 + 1152


def test_results_of_reading_that_overlap_are_refused(lib):  # noqa: F811
    far = 1 << 20
    for key, value in ((0, 0), (0, 16), (0, READ - 16), (READ - 16, 0)):
        refused(lib, read_call(lib, key, value, far, 2 * far), "overlap")
    for k in (0, 1):
        for at in (0, 16, READ - 16, 16 - HELD):
            caches = [2 * far, 3 * far]
            caches[k] = far + at  # with the values' result at `far`
            refused(lib, read_call(lib, 0, far, *caches), "overlap the cache")
            refused(lib, read_call(lib, far, 0, *caches), "overlap the cache")
        caches = [2 * far, 3 * far]
        caches[k] = far + 16 - HELD4[k]
        refused(lib, read_call(lib, 0, far, *caches, **CACHES4), "overlap the cache")


@without_gpu
def test_results_of_reading_beside_each_other_are_taken(lib):  # noqa: F811
    far = 1 << 20
    for args in ((0, READ, far, 2 * far), (READ, 0, far, far), (0, READ, 2 * READ, 2 * READ + HELD), (HELD, HELD + READ, 0, 0)):
        assert read_call(lib, *args) == -2, lib.fbgemm_amd_last_error()
    assert read_call(lib, HELD4[0], HELD4[0] + READ, 0, HELD4[0] + 2 * READ, **CACHES4) == -2, lib.fbgemm_amd_last_error()
    assert read_call(lib, 0, READ, 0, 0, blocks=0) == -2, lib.fbgemm_amd_last_error()
    assert read_call(lib, 0, 0, 0, 0, tokens=0) == 0
