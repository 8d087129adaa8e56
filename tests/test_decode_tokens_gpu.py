"""Rotary positions and sampling against their formulas in 64 bits, and a whole decoding step: positions, 4-bit cache, attention, logits, tokens."""
import math

import numpy as np
import pytest

import decode_tokens_reference as R
from test_decode_finite_gpu import close_and_finite as close
from test_decode_gpu import np64

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


# ---- rotary positions -------------------------------------------------------------------------------


def check_rotation(decode, query, key, positions, frequencies, out=None, **kw):
    held = [np64(query), np64(key)]
    got = decode.rotate_positions(query, key, positions, frequencies, out=out, **kw)
    n = 2 * len(frequencies)
    for x, y, like in zip(got, held, (query, key)):
        want, off = R.rotate(y, positions.cpu().numpy(), frequencies.cpu().numpy(), **kw)
        assert x.dtype == like.dtype and x.shape == like.shape
        close(x, want, off, x.dtype)
        assert np.array_equal(np64(x)[..., n:], y[..., n:])
    return got


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,turned", [
    (1, 1, 1, 2, 2), (5, 4, 2, 64, 64), (64, 32, 8, 128, 128), (33, 3, 3, 80, 32), (7, 2, 1, 96, 48), (3, 5, 2, 30, 20), (2, 3, 1, 8, 0), (9, 2, 2, 7, 6),
    (4, 1, 1, 256, 250), (2, 1, 2, 2100, 2048), (8200, 2, 1, 16, 16), (8193, 1, 1, 10, 4)])
def test_rotation(decode, tokens, heads, kv_heads, dim, turned, dtype, interleaved):
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + dim)
    fused = torch.randn((tokens, heads + 2 * kv_heads, dim), device="cuda", generator=g).to(dtype)
    positions = torch.randint(0, 5000, (tokens,), device="cuda", generator=g, dtype=torch.int32 if dim % 3 else torch.int64)
    f = decode.rotary_frequencies(turned) if turned else torch.zeros(0, dtype=torch.float64, device="cuda")
    query, key = fused[:, :heads], fused[:, heads:heads + kv_heads]
    check_rotation(decode, query, key, positions, f, interleaved=interleaved)
    dense = [query.contiguous(), key.contiguous()]
    got = check_rotation(decode, *dense, positions, f, interleaved=interleaved, magnitude=1.5, inverse=True)
    # over the inputs: the same bits, and nothing beside them
    rest = fused[:, heads + kv_heads:].clone()
    same = decode.rotate_positions(query, key, positions, f, interleaved=interleaved, magnitude=1.5, inverse=True, out=(query, key))
    assert same[0].data_ptr() == query.data_ptr() and torch.equal(query, got[0]) and torch.equal(key, got[1])
    assert torch.equal(fused[:, heads + kv_heads:], rest)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotation_of_rows_off_their_boundaries_and_in_other_orders(decode, dtype, interleaved):
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    wide = torch.randn((20, 6, 70), device="cuda", generator=g).to(dtype)
    positions, f = torch.arange(20, device="cuda") * 7, decode.rotary_frequencies(32)
    a = wide[:, :4, 3:67], wide[:, 4:, 3:67]
    want = check_rotation(decode, *a, positions, f, interleaved=interleaved)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in a]
    got = check_rotation(decode, *heads_first, positions, f, interleaved=interleaved)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = decode.rotate_positions(*heads_first, positions, f, interleaved=interleaved, out=tuple(heads_first))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = a[0][:, :1].expand(-1, 3, -1)  # heads that are one
    got = decode.rotate_positions(one, a[1], positions, f, interleaved=interleaved)
    assert torch.equal(got[0], want[0][:, :1].expand(-1, 3, -1))
    places = torch.zeros((20, 6, 70), dtype=dtype, device="cuda")  # results inside a wider tensor
    got = decode.rotate_positions(*a, positions, f, interleaved=interleaved, out=(places[:, :4, 5:69], places[:, 4:, 5:69]))
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and (places[..., :5] == 0).all() and (places[..., 69:] == 0).all()


def test_rotation_of_far_positions(decode):
    """Angles of 2^31 radians and beyond, and negative ones: what is left of them behind whole turns."""
    positions = torch.tensor([0, 1, 262_143, 2**31 - 1, 2**31 + 5, 2**40 + 12345, -1, -262_143], device="cuda")
    x = torch.randn((8, 3, 64), device="cuda")
    check_rotation(decode, x, x, positions, decode.rotary_frequencies(64))
    check_rotation(decode, x, x, positions, decode.rotary_frequencies(64, factor=8.0, trained=8192), interleaved=True)
    got = decode.rotate_positions(x, x, positions, decode.rotary_frequencies(64))[0]
    assert torch.equal(got[0], x[0])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,tokens", [(torch.bfloat16, 4300), (torch.float16, 4300), (torch.float32, 2150)])
def test_rotation_past_the_caches_gives_the_same_bits(decode, dtype, tokens, interleaved):
    """Results of more than 64 MB, and the same tokens in parts."""
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    q, k = (torch.randn((tokens, n, 128), device="cuda", generator=g).to(dtype) for n in (48, 16))
    positions, f = torch.arange(tokens, device="cuda") * 3, decode.rotary_frequencies(96)
    got = decode.rotate_positions(q, k, positions, f, interleaved=interleaved)
    for part in torch.arange(tokens, device="cuda").split(1000):
        want = decode.rotate_positions(q[part], k[part], positions[part], f, interleaved=interleaved)
        assert all(torch.equal(x[part], y) for x, y in zip(got, want))
    decode.rotate_positions(q, k, positions, f, interleaved=interleaved, out=(q, k))
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])


def test_a_rotations_gradient_is_the_inverse(decode):
    """<R x, y> = <x, R' y> of the linear map, and turning back and forth: a rounding of each of the two turns."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x, y = (torch.randn((50, 4, 64), device="cuda", generator=g) for _ in range(2))
    positions, f = torch.arange(50, device="cuda") * 99, decode.rotary_frequencies(48)
    for interleaved in (False, True):
        there = decode.rotate_positions(x, x, positions, f, interleaved=interleaved, magnitude=1.25)[0]
        back = decode.rotate_positions(y, y, positions, f, interleaved=interleaved, magnitude=1.25, inverse=True)[0]
        a, b = (there.double() * y.double()).sum(), (x.double() * back.double()).sum()
        # both sides: 7 roundings of 2^-24 of every element's product
        assert abs(a - b) <= 14 * 2.0 ** -24 * 1.25 * 2 * (x.double().abs().sum() * y.abs().max())
        # against differences of one element: the map is linear, so any step will do
        bumped = x.clone()
        bumped[7, 2, 5] += 1.0
        step = (decode.rotate_positions(bumped, bumped, positions, f, interleaved=interleaved, magnitude=1.25)[0].double() - there.double())
        assert abs((step * y.double()).sum() - back[7, 2, 5].double()) < 1e-4  # some 64 numbers of 2^-22
        again = decode.rotate_positions(there, there, positions, f, interleaved=interleaved, magnitude=0.8, inverse=True)[0]
        # 0.8 and 1.25 as fp32 numbers, and twice 7 roundings of a pair's two numbers
        assert (again - x).abs().max() <= 16 * 2.0 ** -23 * x.abs().max() * 2


# ---- sampling ---------------------------------------------------------------------------------------


def check_samples(decode, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    cu = lambda a, t: None if a is None else torch.tensor(a, dtype=t, device="cuda")  # noqa: E731
    call = lambda: decode.sample_tokens(logits, cu(uniform, torch.float32), cu(temperature, torch.float32), cu(top_k, torch.int32),  # noqa: E731
                                        cu(top_p, torch.float32), cu(min_p, torch.float32))
    got = call()
    again = call()
    assert torch.equal(got.tokens, again.tokens) and torch.equal(got.log_probabilities, again.log_probabilities)
    assert got.tokens.dtype == torch.int64 and got.log_probabilities.dtype == torch.float32
    x = np64(logits)
    of = lambda a, r, none: none if a is None else float(np.float32(a[r]))  # noqa: E731
    for r, (token, logp) in enumerate(zip(got.tokens.tolist(), got.log_probabilities.tolist())):
        s = R.Sampled(x[r], of(temperature, r, 1.0), 0 if top_k is None else top_k[r], of(top_p, r, 1.0), of(min_p, r, 0.0))
        assert s.holds(token, np.float32(uniform[r]), logp), (r, token, logp, uniform[r], s.empty or (s.order[:5], s.w[:5], s.sure, len(s.order)))
    return got


def rows_of(seed, rows, vocab, dtype, spread=3.0, gone=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = spread * torch.randn((rows, vocab), device="cuda", generator=g)
    x.masked_fill_(torch.rand((rows, vocab), device="cuda", generator=g) < gone, -math.inf)
    return x.to(dtype)


VOCABS = [1, 2, 3, 7, 8, 9, 63, 65, 500, 4095, 4096, 8193, 32_000, 65_536, 65_537, 131_071, 131_072, 131_073, 200_001, 1 << 20]
FILTERS = {
    "none": {}, "temperature": dict(temperature=[0.3, 0.0, 1.0, 2.5, 0.9, -1.0]), "top_k": dict(top_k=[1, 5, 0, 50, 1000, -3]), "top_p": dict(top_p=[0.5, 0.9, 1.0, 0.99, 0.1, 0.0]),
    "min_p": dict(min_p=[0.1, 0.0, 0.5, 1.0, 0.01, -1.0]),
    "all": dict(temperature=[0.7, 1.0, 1.5, 0.5, 1.0, 0.8], top_k=[40, 0, 100, 1500, 0, 7], top_p=[0.9, 0.95, 1.0, 0.8, 1.0, 0.6], min_p=[0.05, 0.0, 0.1, 0.0, 0.02, 0.0])}


@pytest.mark.parametrize("filters", list(FILTERS))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_samples(decode, vocab, dtype, filters):
    rng = np.random.default_rng(vocab)
    check_samples(decode, rows_of(vocab, 6, vocab, dtype), rng.uniform(0, 1, 6).tolist(), **FILTERS[filters])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,top_k", [(5000, 1023), (5000, 1024), (5000, 1025), (5000, 4999), (5000, 5000), (5000, 9000), (100_000, 60_000), (300_000, 2000), (300_000, 100)])
def test_the_first_k_at_the_limits_of_k(decode, vocab, top_k, dtype):
    rng = np.random.default_rng(top_k)
    check_samples(decode, rows_of(top_k, 4, vocab, dtype), rng.uniform(0, 1, 4).tolist(), top_k=[top_k] * 4)
    check_samples(decode, rows_of(top_k, 4, vocab, dtype, gone=0.99), rng.uniform(0, 1, 4).tolist(), top_k=[top_k] * 4, top_p=[0.9, 0.5, 1.0, 0.99])


@pytest.mark.parametrize("filters", list(FILTERS))
@pytest.mark.parametrize("vocab", [9, 5000, 140_000])
def test_samples_of_logits_many_of_which_are_equal(decode, vocab, filters):
    """Equal logits are in the order of their tokens: which of them are within k or p is exact."""
    rng = np.random.default_rng(vocab)
    for grid in (1.0, 8.0):
        x = torch.round(rows_of(vocab, 6, vocab, torch.float32) / grid) * grid
        check_samples(decode, x, rng.uniform(0, 1, 6).tolist(), **FILTERS[filters])
        check_samples(decode, x.bfloat16(), rng.uniform(0, 1, 6).tolist(), **FILTERS[filters])
    flat = torch.full((6, vocab), -0.0, device="cuda")
    flat[:, ::2] = 0.0  # zeros of both signs are equal
    check_samples(decode, flat, [0.0, 0.2, 0.4, 0.6, 0.8, 0.999], **FILTERS[filters])


def test_the_lowest_of_equal_tokens_come_first(decode):
    x = torch.zeros((4, 3000), device="cuda")
    x[:, ::3] = 1.0  # tokens 0, 3, ..., 2997 are the most likely
    got = decode.sample_tokens(x, torch.full((4,), 0.9999, device="cuda"), top_k=torch.tensor([5, 1000, 1001, 1], device="cuda", dtype=torch.int32))
    assert got.tokens.tolist() == [12, 2997, 2997, 0]
    assert torch.allclose(got.log_probabilities, torch.tensor([math.log(1 / 5), math.log(1 / 1000), math.log(math.e / (1000 * math.e + 1)), 0.0], device="cuda"))
    got = decode.sample_tokens(x, torch.full((4,), 0.9999, device="cuda"), temperature=torch.tensor([0.0, 1.0, 1.0, float("nan")], device="cuda"),
                               top_p=torch.tensor([1.0, 0.0, 1e-9, 1.0], device="cuda"))
    assert got.tokens.tolist() == [0, 0, 0, 0] and (got.log_probabilities == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_samples_of_masked_rows_and_of_numbers_that_are_not_finite(decode, dtype):
    x = rows_of(3, 8, 9000, dtype, gone=0.5)
    x[0] = -math.inf                     # nothing is left
    x[1] = float("nan")
    x[2, :] = -math.inf
    x[2, 8999] = torch.finfo(dtype).min  # one token, of the type's lowest value
    x[3, ::2] = float("nan")
    x[4, 77], x[4, 8000] = math.inf, math.inf
    x[5] = -math.inf
    x[5, 4000:4003] = torch.tensor([-5.0, 1.0, 2.0]).to(dtype)
    x[6] = torch.finfo(dtype).min        # a mask of the type's lowest value
    x[6, 123] = 1.0
    x[7] = torch.finfo(dtype).min
    u = [0.3, 0.3, 0.3, 0.7, 0.7, 0.5, 0.5, 0.25]
    for filters in ({}, dict(top_k=[4] * 8), dict(top_p=[0.7] * 8), dict(min_p=[0.2] * 8), dict(top_k=[2000] * 8, top_p=[0.7] * 8, min_p=[0.2] * 8, temperature=[0.8] * 8)):
        got = check_samples(decode, x, u, **filters)
        assert got.tokens[:3].tolist() == [-1, -1, 8999] and int(got.tokens[4]) in (77, 8000) and int(got.tokens[6]) == 123
    got = check_samples(decode, x, u, temperature=[0.0] * 8)
    assert got.tokens.tolist()[4:7] == [77, 4002, 123] and got.tokens.tolist()[:3] == [-1, -1, 8999] and int(got.tokens[7]) == 0


def test_uniform_numbers_and_temperatures_at_their_ends(decode):
    x = rows_of(5, 9, 5000, torch.float32)
    u = [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), 2.0 ** -149, 0.5, 0.5]
    check_samples(decode, x, u)
    check_samples(decode, x, u, top_k=[10] * 9, top_p=[0.9] * 9)
    check_samples(decode, x, u, temperature=[1e-30, 1e-38, 1e-45, 1e30, float("inf"), 1e-3, 100.0, 3e38, 1.0])
    check_samples(decode, x, u, temperature=[1e-30, 1e-38, 1e-45, 1e30, float("inf"), 1e-3, 100.0, 3e38, 1.0], top_k=[100] * 9, top_p=[0.5] * 9, min_p=[0.9] * 9)


def test_samples_of_logits_as_far_apart_as_numbers_are(decode):
    """Their difference is beyond fp32, and a high temperature lets all of them weigh the same."""
    for vocab in (6000, 40_000):
        x = rows_of(8, 6, vocab, torch.float32) * 2e37
        u = [0.0, 0.2, 0.4, 0.6, 0.8, 0.99]
        for t in (1e38, 3e38, float("inf")):
            check_samples(decode, x, u, temperature=[t] * 6, top_p=[0.5, 0.9, 0.1, 0.99, 1.0, 0.3])
            check_samples(decode, x.bfloat16(), u, temperature=[t] * 6, top_p=[0.5, 0.9, 0.1, 0.99, 1.0, 0.3], min_p=[0.0, 0.3, 0.9, 0.0, 0.5, 0.99])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [8191, 8192, 20_001, 32_768, 32_769])
def test_samples_of_more_rows_than_the_device_has_compute_units(decode, vocab, dtype):
    rows = 300
    rng = np.random.default_rng(vocab)
    pick = lambda *of: rng.choice(of, rows).tolist()  # noqa: E731
    check_samples(decode, rows_of(vocab, rows, vocab, dtype), rng.uniform(0, 1, rows).tolist(), temperature=pick(1.0, 0.0, 0.6, 1.4), top_k=pick(0, 0, 0, 50, 3000),
                  top_p=pick(1.0, 1.0, 0.9, 0.99), min_p=pick(0.0, 0.0, 0.05))


def test_samples_of_strided_shared_and_many_rows(decode):
    wide = rows_of(6, 5, 9050, torch.bfloat16)
    u = [0.1, 0.3, 0.5, 0.7, 0.9]
    check_samples(decode, wide[:, 13:9014], u, top_p=[0.9] * 5)
    check_samples(decode, wide[:1, 1:8000].expand(5, -1), u, top_k=[100] * 5)
    check_samples(decode, wide[::2, :100], u[:3])
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn((70_000, 3), device="cuda", generator=g)
    uniform = torch.rand(70_000, device="cuda", generator=g)
    got = decode.sample_tokens(x, uniform)
    p = torch.softmax(x.double(), -1)
    want = (p.cumsum(-1) <= uniform.double()[:, None]).sum(-1)
    assert torch.equal(got.tokens, want)  # no number of the 70 000 is within 2^-40 of a border
    assert (got.log_probabilities.double() - torch.log(p.gather(1, want[:, None])[:, 0])).abs().max() < 2.0 ** -20
    assert decode.sample_tokens(x[:0], uniform[:0]).tokens.shape == (0,)


def test_how_often_tokens_are_drawn(decode):
    """65 536 numbers spread evenly over [0, 1): a token of probability p is drawn p times as often, to one draw at either end."""
    n = 1 << 16
    x = rows_of(8, 1, 50, torch.float32, spread=1.0)
    uniform = torch.arange(n, device="cuda").float() / n
    got = decode.sample_tokens(x.expand(n, -1), uniform, top_k=torch.full((n,), 20, device="cuda", dtype=torch.int32))
    top = torch.topk(x[0].double(), 20)
    p = torch.zeros(50, device="cuda", dtype=torch.float64).index_copy_(0, top.indices, torch.softmax(top.values, 0))
    count = torch.bincount(got.tokens, minlength=50)
    assert (count - p * n).abs().max() <= 1 and (count[p == 0] == 0).all()


# ---- together ---------------------------------------------------------------------------------------


def step(decode, s):
    t = decode.kv_block_tables(s["lengths"], s["new"], s["tables"], s["free"], s["start"], 16, len(s["qkv"]))
    query, key = decode.rotate_positions(s["qkv"][:, :8], s["qkv"][:, 8:10], t.positions, s["frequencies"])
    decode.kv_cache_append(key, s["qkv"][:, 10:], s["kc"], s["vc"], t.slots, row_bits=4)
    out, lse = decode.paged_attention(query, s["kc"], s["vc"], s["tables"], t.lengths, row_bits=4)
    rows = decode.kv_cache_read(s["kc"], s["vc"], s["tables"], s["offsets"], 500, 64, torch.bfloat16, row_bits=4)
    logits = decode.penalize_logits(s["logits"] + out.flatten(1)[:, :1], s["said"], s["said_offsets"], frequency=s["frequency"])
    tokens, log_p = decode.sample_tokens(logits, s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return (*t, query, key, out, lse, *rows, tokens, log_p, s["kc"].clone(), s["vc"].clone())


def step_state(decode, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B = 5
    lengths = torch.tensor([0, 16, 31, 300, 77], device="cuda", dtype=torch.int32)[torch.randperm(B, device="cuda", generator=g)]
    pages = torch.randperm(60, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((B, 24), -1, dtype=torch.int32, device="cuda")
    used = (lengths + 15) // 16
    tables[torch.arange(24, device="cuda") < used[:, None]] = pages[: int(used.sum())]
    rand = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
    s = dict(lengths=lengths, new=torch.ones_like(lengths), tables=tables, free=pages, start=used.sum().to(torch.int32).reshape(1),
             qkv=torch.randn((B, 12, 64), device="cuda", generator=g).bfloat16(), logits=2 * torch.randn((B, 4000), device="cuda", generator=g),
             said=torch.randint(0, 4000, (100,), device="cuda", generator=g), said_offsets=torch.arange(B + 1, device="cuda") * 20, frequency=rand(B),
             uniform=rand(B), temperature=0.5 + rand(B), top_k=torch.tensor([0, 5, 50, 2000, 1], device="cuda", dtype=torch.int32), top_p=0.5 + 0.5 * rand(B),
             min_p=0.1 * rand(B), frequencies=decode.rotary_frequencies(64), offsets=torch.zeros(B + 1, device="cuda", dtype=torch.int32))
    s["offsets"][1:] = (lengths + 1).cumsum(0)
    for name in ("kc", "vc"):
        s[name] = torch.randint(0, 60, (60, 2, 16, 36), device="cuda", generator=g, dtype=torch.uint8)
    return s


def test_a_captured_step_replays_and_follows_its_inputs(decode):
    s = step_state(decode, 1)
    others = [step_state(decode, k) for k in (2, 3, 4, 5)]
    step(decode, {k: v.clone() for k, v in s.items()})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(decode, s)
    for o in others:
        want = step(decode, {k: v.clone() for k, v in o.items()})
        torch.cuda.synchronize()
        for k, v in s.items():
            v.copy_(o[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (got[-4] >= 0).all() and torch.isfinite(got[7]).all()


def test_a_step_on_another_stream(decode):
    s = step_state(decode, 5)
    want = step(decode, {k: v.clone() for k, v in s.items()})
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:
        with torch.cuda.stream(side):
            got.append(step(decode, {k: v.clone() for k, v in s.items()}))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_rows_that_are_read_back_are_the_ones_attention_sees(decode):
    """Attention over a cache of 16-bit rows that hold what the 4-bit ones stand for: the same to the values' rounding to 16 bits
    (2^-9 of each, their differences average out: twice that of the largest) and the scores' (128 products of 2^-9, by the scale)."""
    s = step_state(decode, 7)
    out, lse = decode.paged_attention(s["qkv"][:, :8], s["kc"], s["vc"], s["tables"], s["lengths"], row_bits=4)
    offsets = torch.zeros(6, device="cuda", dtype=torch.int32)
    offsets[1:] = s["lengths"].cumsum(0)
    n = int(offsets[-1])
    key, value = decode.kv_cache_read(s["kc"], s["vc"], s["tables"], offsets, n, 64, row_bits=4)
    for r in range(5):
        k, v = (x[offsets[r]:offsets[r + 1]].double().transpose(0, 1) for x in (key, value))
        q = s["qkv"][r, :8].double().view(2, 4, 64)
        if k.shape[1] == 0:
            assert (out[r] == 0).all()
            continue
        scores = (q[:, :, None] * k[:, None]).sum(-1) / 8
        want = (torch.softmax(scores, -1)[..., None] * v[:, None]).sum(2).view(8, 64)
        # one rounding to bf16, and what fp32 leaves of the terms' sizes
        assert (out[r].double() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + 2.0 ** -12 * v.abs().max()
        assert (lse[r].double() - torch.logsumexp(scores, -1).view(8)).abs().max() < 2.0 ** -12 * (1 + scores.abs().max())


def test_refusals(decode):
    s = step_state(decode, 6)
    f, p = s["frequencies"], torch.arange(5, device="cuda")
    q, k = s["qkv"][:, :8], s["qkv"][:, 8:10]
    rotate = lambda query=q, key=k, positions=p, frequencies=f, **kw: decode.rotate_positions(query, key, positions, frequencies, **kw)  # noqa: E731
    sample = lambda logits=s["logits"], uniform=s["uniform"], **kw: decode.sample_tokens(logits, uniform, **kw)  # noqa: E731
    refused = [
        lambda: rotate(query=q.float()), lambda: rotate(query=q.double(), key=k.double()), lambda: rotate(query=q[:4]), lambda: rotate(query=q[0], key=k[0]),
        lambda: rotate(query=q[..., :60]), lambda: rotate(positions=p.float()), lambda: rotate(positions=p[:4]), lambda: rotate(positions=p.cpu()),
        lambda: rotate(frequencies=f.float()), lambda: rotate(frequencies=torch.ones(33, device="cuda", dtype=torch.float64)), lambda: rotate(frequencies=f.cpu()),
        lambda: rotate(frequencies=f.view(2, 16)), lambda: rotate(magnitude=float("inf")), lambda: rotate(query=q.transpose(1, 2), key=k.transpose(1, 2)),
        lambda: rotate(query=torch.zeros((5, 1, 2200), device="cuda"), key=torch.zeros((5, 1, 2200), device="cuda"), frequencies=torch.ones(1100, device="cuda", dtype=torch.float64)),
        lambda: rotate(out=(q, q[:, :2])), lambda: rotate(out=(s["qkv"][:, 1:9], k)), lambda: rotate(out=(q, s["qkv"][:, 9:11])), lambda: rotate(out=(q.float(), k)),
        lambda: rotate(out=(k, q)), lambda: rotate(out=(q[:, :1].expand(-1, 8, -1), k)),
        lambda: sample(logits=s["logits"].double()), lambda: sample(logits=s["logits"][0]), lambda: sample(logits=s["logits"].t()), lambda: sample(logits=s["logits"][:, :0]),
        lambda: sample(uniform=s["uniform"][:4]), lambda: sample(uniform=s["uniform"].double()), lambda: sample(uniform=s["uniform"].cpu()),
        lambda: sample(temperature=s["temperature"][:3]), lambda: sample(top_k=s["top_k"].long()), lambda: sample(top_p=s["top_p"].half()), lambda: sample(min_p=s["min_p"].cpu()),
        lambda: sample(logits=torch.zeros((1, (1 << 20) + 1), device="cuda"), uniform=s["uniform"][:1]),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError, TypeError, NotImplementedError)):
            call()
            print("not refused:", i)
    step(decode, s)
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError):  # no CPU path
        decode.sample_tokens(s["logits"].cpu(), s["uniform"].cpu())


@pytest.mark.parametrize("rows, rotary, temperature", [(16, True, 0.0), (16, True, 0.8), (4, False, 0.0), (4, True, 0.8), (8, True, 1.5)])
def test_the_example_runs_with_positions_4_bit_rows_and_draws(decode, rows, rotary, temperature):
    """Logits of the paged path against the dense layer. 16-bit rows: attention's outputs round to bf16 in both, as queries and keys that were turned
    do. A row of 64 normal numbers has a range of some 5 standard deviations: codes of 8 bits are off by 5 / 255 / sqrt(12) = 0.006 of one, of 4
    bits by 0.1. A score, of standard deviation 1, and so a weight is off by as much, and an output by both: 0.14 in 4 bits; twice that
    for the worst of a few requests."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    said, lengths, logits, d = example.generate(requests=5, steps=20, rows8=rows == 8, rows4=rows == 4, rotary=rotary, temperature=temperature)
    for r in range(5):
        n = int(lengths[r])
        assert (said[r, :n] >= 0).all() and (said[r, n:] == -1).all()
        want = example.dense_logits(d, said[r, :n - 1]).float()
        assert float((logits[r].float() - want).norm() / want.norm()) < {16: 0.02, 8: 0.05, 4: 0.28}[rows]
