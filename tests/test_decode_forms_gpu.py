"""Forms of the decoding step's operators that a program may use and that no other file here runs: layouts, gradients, extremes."""
import numpy as np
import pytest

import decode_tokens_reference as R
import test_decode_rows4_gpu as A
from test_decode_finite_gpu import close_and_finite as close
from test_decode_gpu import np64
from test_decode_tokens_gpu import TYPES, check_rotation

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 33])
def test_rotation_of_heads_whose_parts_are_side_by_side(decode, tokens, dtype, interleaved):
    """A projection [tokens, heads, 3, dim], turned in place, and results put into such a buffer."""
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    x = torch.randn((tokens, 8, 3, 64), device="cuda", generator=g).to(dtype)
    query, key, value = x.unbind(2)
    positions, f = torch.arange(tokens, device="cuda") * 5, decode.rotary_frequencies(64)
    want = check_rotation(decode, query, key, positions, f, interleaved=interleaved)
    held = value.clone()
    places = torch.zeros_like(x)
    got = decode.rotate_positions(query, key, positions, f, interleaved=interleaved, out=(places[:, :, 0], places[:, :, 2]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (places[:, :, 1] == 0).all()
    decode.rotate_positions(query, key, positions, f, interleaved=interleaved, out=(query, key))
    assert torch.equal(query, want[0]) and torch.equal(key, want[1]) and torch.equal(value, held)


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_a_rotation(decode, dtype, interleaved, inverse):
    """Of a fused projection's parts, through autograd: the formula's in 64 bits, and differences of single elements."""
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    fused = normal(40, 12, 64).to(dtype).requires_grad_()
    positions, f = torch.randint(0, 5000, (40,), device="cuda", generator=g), decode.rotary_frequencies(48)
    kw = dict(interleaved=interleaved, magnitude=1.25, inverse=inverse)
    query, key = decode.rotate_positions(fused[:, :8], fused[:, 8:10], positions, f, **kw)
    back = [normal(40, 8, 64).to(dtype), normal(40, 2, 64).to(dtype)]
    got, = torch.autograd.grad((query, key), fused, back)
    for k, part in enumerate((slice(0, 8), slice(8, 10))):
        want, off = R.rotate(np64(back[k]), positions.cpu().numpy(), f.cpu().numpy(), interleaved, 1.25, inverse=not inverse)
        close(got[:, part], want, off, dtype)
    assert (got[:, 10:] == 0).all()
    # against differences: the map is linear, so a step of one will do; fp32 numbers, some 64 products of 2^-21
    if dtype == torch.float32:
        with torch.no_grad():
            for t, h, d in ((3, 1, 5), (39, 9, 40), (0, 8, 63)):
                there = fused.detach().clone()
                there[t, h, d] += 1.0
                a, b = decode.rotate_positions(there[:, :8], there[:, 8:10], positions, f, **kw)
                change = ((a.double() - query.double()) * back[0]).sum() + ((b.double() - key.double()) * back[1]).sum()
                assert abs(float(change) - float(got[t, h, d])) < 64 * 2.0 ** -21 * 16
    # only one of the two, gradients that are one number for all, and a gradient's gradient
    q = normal(40, 8, 64).to(dtype).requires_grad_()
    decode.rotate_positions(q, fused[:, 8:10].detach(), positions, f, **kw)[0].sum().backward()
    want, off = R.rotate(np64(torch.ones_like(q)), positions.cpu().numpy(), f.cpu().numpy(), interleaved, 1.25, inverse=not inverse)
    close(q.grad, want, off, dtype)
    v = back[0].clone().requires_grad_()
    first, = torch.autograd.grad(decode.rotate_positions(q, q, positions, f, **kw)[0], q, v, create_graph=True)
    w = normal(40, 8, 64).to(dtype)
    second, = torch.autograd.grad(first, v, w)
    want, off = R.rotate(np64(w), positions.cpu().numpy(), f.cpu().numpy(), interleaved, 1.25, inverse=inverse)
    close(second, want, off, dtype)
    # on another stream, whose backward runs there too
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, = torch.autograd.grad(decode.rotate_positions(fused[:, :8], fused[:, 8:10], positions, f, **kw), fused, back)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, got)


def test_given_tensors_that_a_graph_follows_are_refused(decode):
    x = torch.randn((5, 12, 64), device="cuda", requires_grad=True) * 1
    q, k, p, f = x[:, :8], x[:, 8:10], torch.arange(5, device="cuda"), decode.rotary_frequencies(64)
    held = x.detach().clone()
    for call in (lambda: decode.rotate_positions(q, k, p, f, out=(q, k)), lambda: decode.rotate_positions(q.detach(), k.detach(), p, f, out=(q, k))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    assert torch.equal(x, held)
    with torch.no_grad():
        decode.rotate_positions(q, k, p, f, out=(q, k))
    assert not torch.equal(x, held)


def large_case(decode, dim, power, dtype, down, block=16):
    """Queries of up to 2^power, and keys that are 2^-down of attention_case's."""
    query, caches, tables, lengths = A.attention_case(decode, dim, dim, 4, 2, block, [1, 33, 200], dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(power)
    query = ((2 * torch.rand(query.shape, device="cuda", generator=g, dtype=torch.float64) - 1) * 2.0 ** power).clamp(-float(torch.finfo(dtype).max), float(torch.finfo(dtype).max)).to(dtype)
    pair = caches[0][..., :4].clone().view(torch.float16)
    caches[0][..., :4] = (pair.float() * 2.0 ** -down).half().view(torch.uint8)
    return query, caches, tables, lengths


def one_token_each(case, scale):
    """Where the largest score is so far above the next one, rounded however, that its token's value is the output: which, and that value."""
    query, caches, tables, lengths = case
    B, Hq, D = query.shape
    H, S = caches[0].shape[1:3]
    hosts, q = [c.cpu().numpy() for c in caches], np64(query)
    sure, value = np.zeros((B, Hq), bool), np.zeros((B, Hq, D))
    for r, n in enumerate(lengths.tolist()):
        at = lambda c, h: c[tables[r].cpu().numpy()[np.arange(n) // S], h, np.arange(n) % S]  # noqa: E731
        for h in range(Hq):
            k, v = (R.rows4_values(at(c, h // (Hq // H)), D) for c in hosts)
            s, wrong = scale * (k @ q[r, h]), (D + 8) * 2.0 ** -22 * abs(scale) * 15 * (np.abs(k).max(0) @ np.abs(q[r, h]))
            order = np.argsort(s)
            sure[r, h] = n == 1 or s[order[-1]] - s[order[-2]] > 2 * wrong + 100
            value[r, h] = v[order[-1]]
    return sure, value


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", [16, 10])
@pytest.mark.parametrize("power", [10, 20, 26, 30, 40, 60])
def test_attention_over_4_bit_rows_of_large_scores(decode, power, block, dtype):
    """Scores of 2^power and beyond: their differences are what weights are made of, however large they are themselves."""
    case = large_case(decode, 128, 0, dtype, 0, block)
    A.check(decode, case, dtype, scale=2.0 ** power)
    A.check(decode, case, dtype, scale=-2.0 ** power, window=40)
    if power >= 20:
        out, lse = decode.paged_attention(case[0], *case[1], *case[2:], scale=2.0 ** power, row_bits=4)
        sure, value = one_token_each(case, 2.0 ** power)
        assert sure.mean() > 0.8
        near = 2.0 ** -15 * 30 * np.abs(value).max() + torch.finfo(dtype).eps * np.abs(value)
        assert (np.abs(np64(out) - value) <= near)[sure].all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [90, 100, 117, 119, 122, 125, 127])
def test_attention_over_4_bit_rows_of_queries_near_the_types_largest(decode, power, dim):
    """The logarithm of the sum is the largest score there, up to 2^112, and one token's value the output."""
    case = large_case(decode, dim, power, torch.bfloat16, 18)
    A.check(decode, case, torch.bfloat16)
    out, lse = decode.paged_attention(case[0], *case[1], *case[2:], row_bits=4)
    assert lse.abs().max() > 2.0 ** (power - 24)
    sure, value = one_token_each(case, dim ** -0.5)
    assert sure.mean() > 0.8
    # weights of 16 bits, a rounding to bf16, and codes up to 15 in sums of fp32
    near = 2.0 ** -15 * 30 * np.abs(value).max() + torch.finfo(torch.bfloat16).eps * np.abs(value)
    assert (np.abs(np64(out) - value) <= near)[sure].all()
    A.check(decode, case, torch.bfloat16, softcap=2.0 ** (power - 20))  # caps that leave most scores a slope
    A.check(decode, case, torch.bfloat16, scale=-dim ** -0.5, window=17)


@pytest.mark.parametrize("power", [80, 100, 110])
def test_attention_over_4_bit_rows_with_large_scales(decode, power):
    for dtype in (torch.float16, torch.bfloat16):
        case = large_case(decode, 128, 0, dtype, 4)
        A.check(decode, case, dtype, scale=2.0 ** power)
        A.check(decode, case, dtype, scale=-2.0 ** power, softcap=2.0 ** (power - 3))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_over_caches_whose_pages_are_differently_far_apart(decode, dim, bits, dtype):
    """Value pages beside something else, key pages behind each other, and the other way round: the same bits as of caches alike."""
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    row = decode.kv_row_bytes(dim, bits)
    caches = [torch.randint(0, 256, (60, 2, 32, row), device="cuda", generator=g, dtype=torch.uint8) for _ in "kv"]
    for c in caches:
        c[..., :4] = torch.randn((60, 2, 32, 2), device="cuda", generator=g).half().view(torch.uint8)
    tables = torch.randperm(60, device="cuda", generator=g).to(torch.int32).view(3, 20)
    lengths = torch.tensor([1, 333, 640], device="cuda")
    query = torch.randn((3, 8, dim), device="cuda", generator=g).to(dtype)
    want = decode.paged_attention(query, *caches, tables, lengths, row_bits=bits)
    for k in range(2):
        apart = list(caches)
        apart[k] = torch.full((60, 3, 32, row), 255, device="cuda", dtype=torch.uint8)[:, 1:]  # beside rows of NaN
        apart[k].copy_(caches[k])
        got = decode.paged_attention(query, *apart, tables, lengths, row_bits=bits)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isfinite(want[0]).all()


def test_reading_back_by_offsets_and_starts_at_the_ends_of_64_bits(decode):
    """Tokens of such requests have no page: zeros, and the first one's number in the status block."""
    from fbgemm_amd import ops
    c = torch.randint(1, 100, (6, 2, 16, 36), device="cuda", dtype=torch.uint8)
    tables = torch.arange(6, device="cuda", dtype=torch.int32).view(2, 3)
    least, most = -2 ** 63, 2 ** 63 - 1
    st = ops.Status()
    for offsets, starts in (((least, 3, 9), (0, 0)), ((least, 3, 9), (5, 0)), ((least + 1, 3, 9), (47, 0)), ((-2 ** 62, 3, 9), (47, 0)), ((0, 3, 9), (most, 0)),
                            ((0, 3, 9), (least, 0)), ((-most, 3, 9), (most, 0)), ((-2 ** 32 + 3, 3, 9), (-2 ** 32, 0))):
        st.clear()
        at = lambda v: torch.tensor(v, device="cuda")  # noqa: E731
        key, value = decode.kv_cache_read(c, c, tables, at(offsets), 9, 64, starts=at(starts), status=st, row_bits=4)
        want = torch.from_numpy(R.rows4_values(c[3].cpu().numpy(), 64)).float().cuda().transpose(0, 1)
        assert (key[:3] == 0).all() and torch.equal(key[3:], want[:6]) and torch.equal(value, key)
        assert st.read() == (1, 0)


# ---- more work than one launch has workgroups for ----------------------------------------------------


def test_rotation_of_more_tokens_than_workgroups(decode):
    tokens = (1 << 22) + 5
    x = torch.randn((tokens, 2, 8), device="cuda").bfloat16()
    positions, f = torch.arange(tokens, device="cuda"), decode.rotary_frequencies(8)
    got = decode.rotate_positions(x[:, :1], x[:, 1:], positions, f)
    for part in (slice(0, 9), slice((1 << 22) - 4, None)):
        want = check_rotation(decode, x[part, :1], x[part, 1:], positions[part], f)
        assert torch.equal(got[0][part], want[0]) and torch.equal(got[1][part], want[1])


@pytest.mark.parametrize("bits", [16, 4])
def test_reading_back_of_more_tokens_than_workgroups(decode, bits):
    tokens = (1 << 24) + 77
    blocks = -(-tokens // 16)
    if bits == 16:
        c = torch.randn((blocks, 1, 16, 8), device="cuda").bfloat16()
    else:
        c = torch.randint(0, 256, (blocks, 1, 16, decode.kv_row_bytes(8, 4)), device="cuda", dtype=torch.uint8)
        c[..., :4] = torch.randn((blocks, 1, 16, 2), device="cuda").half().view(torch.uint8)
    tables = torch.randperm(blocks, device="cuda").int()[None]
    at = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    kw = dict(dtype=torch.bfloat16, row_bits=8 if bits == 16 else 4)
    key, value = decode.kv_cache_read(c, c, tables, at(0, tokens), tokens, 8, **kw)
    assert torch.equal(key, value)
    if bits == 16:
        assert torch.equal(key, c[tables[0].long(), 0].view(-1, 1, 8)[:tokens])
    for first, n in ((0, 50), ((1 << 24) - 40, 117)):
        want = decode.kv_cache_read(c, c, tables, at(0, n), n, 8, starts=at(first), **kw)
        assert torch.equal(key[first:first + n], want[0])


@pytest.mark.parametrize("shift", [0, 1])
def test_append_of_more_rows_than_workgroups(decode, shift):
    """4-bit rows of 8: a lane a row, 256 rows a workgroup and 8 192 of those."""
    from fbgemm_amd import ops
    tokens = 8192 * 256 + 300
    new = torch.randn((tokens, 1, 16), device="cuda").bfloat16()[..., shift:shift + 8]
    kc, vc = (torch.zeros((tokens // 4, 1, 4, 8), device="cuda", dtype=torch.uint8) for _ in "kv")
    slots = torch.randperm(tokens, device="cuda")
    decode.kv_cache_append(new, -new, kc, vc, slots, row_bits=4)
    for c, x in ((kc, new), (vc, -new)):
        want = ops.quantize_rowwise(x.float().reshape(-1, 8), 4, layout=ops.QLAYOUT_TBE)
        assert torch.equal(c.view(tokens, 8)[slots], want)


def test_samples_of_more_rows_than_a_launch_takes(decode):
    """Rows of one launch have fewer than 2^32 threads, 1 024 of them a row; all rows have the same logits."""
    rows = (1 << 22) + 9
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = (3 * torch.randn((1, 33_000), device="cuda", generator=g)).bfloat16()
    uniform = torch.rand(rows, device="cuda", generator=g)
    top_k = torch.randint(1, 40, (rows,), device="cuda", generator=g, dtype=torch.int32)
    got = decode.sample_tokens(x.expand(rows, -1), uniform, top_k=top_k)
    for part in (slice(0, 99), slice((1 << 22) - 50, None)):
        want = decode.sample_tokens(x.expand(len(uniform[part]), -1), uniform[part], top_k=top_k[part])
        assert torch.equal(got.tokens[part], want.tokens) and torch.equal(got.log_probabilities[part], want.log_probabilities)
    assert (got.tokens >= 0).all()


# ---- what refusals say --------------------------------------------------------------------------------


def test_refusals_name_what_they_refuse(decode):
    z = lambda *shape, t=torch.bfloat16: torch.zeros(shape, device="cuda", dtype=t)  # noqa: E731
    q, k, p, f = z(5, 8, 64), z(5, 2, 64), torch.arange(5, device="cuda"), decode.rotary_frequencies(64)
    rotate = lambda query=q, key=k, positions=p, frequencies=f, **kw: decode.rotate_positions(query, key, positions, frequencies, **kw)  # noqa: E731
    logits, uniform = z(5, 100), z(5, t=torch.float32)
    sample = lambda x=logits, u=uniform, **kw: decode.sample_tokens(x, u, **kw)  # noqa: E731
    u8 = lambda *shape: z(*shape, t=torch.uint8)  # noqa: E731
    c4, c16, tables, offsets = u8(4, 2, 16, 36), z(4, 2, 16, 64), z(3, 2, t=torch.int32), torch.arange(4, device="cuda")
    read = lambda kc=c4, vc=c4, t=tables, o=offsets, n=3, dim=64, dtype=None, bits=4, **kw: decode.kv_cache_read(kc, vc, t, o, n, dim, dtype, row_bits=bits, **kw)  # noqa: E731
    append = lambda key=z(3, 2, 64), kc=c4, vc=u8(4, 2, 16, 36), bits=4: decode.kv_cache_append(key, key, kc, vc, torch.arange(3, device="cuda"), row_bits=bits)  # noqa: E731
    attend = lambda query=z(3, 4, 64), kc=c4, vc=c4, bits=4: decode.paged_attention(query, kc, vc, tables, offsets[1:], row_bits=bits)  # noqa: E731
    refused = [
        (lambda: rotate(query=q.float()), "of one type"), (lambda: rotate(query=q.double(), key=k.double()), "float32, float16 or bfloat16"), (lambda: rotate(query=q[:4]), "of one type"),
        (lambda: rotate(positions=p.float()), "positions must be int32 or int64"), (lambda: rotate(positions=p[:4]), "positions must hold 5"), (lambda: rotate(positions=p.cpu()), "positions must be on"),
        (lambda: rotate(frequencies=f.float()), "frequencies must be Double"), (lambda: rotate(frequencies=torch.ones(33, device="cuda", dtype=torch.float64)), "33 frequencies"),
        (lambda: rotate(magnitude=float("inf")), "magnitude must be finite"), (lambda: rotate(query=z(5, 64, 8).transpose(1, 2), key=z(5, 64, 2).transpose(1, 2)), "next to each other"),
        (lambda: rotate(out=(q, q[:, :2])), "must not overlap"), (lambda: rotate(out=(q, k[:, :1].expand(-1, 2, -1))), "rows of a result must not overlap"),
        (lambda: rotate(out=(q.float(), k)), "shapes and type of query and key"), (lambda: rotate(out=(q[:, :, :63], k)), "shapes and type of query and key"),
        (lambda: sample(x=logits.double()), "float32, float16 or bfloat16"), (lambda: sample(x=logits[0]), r"logits must be \[rows, vocab\]"), (lambda: sample(x=z(100, 5).t()), "next to each other"),
        (lambda: sample(x=logits[:, :0]), "vocab must be in 1"), (lambda: sample(u=uniform[:4]), "uniform must hold 5"), (lambda: sample(u=uniform.double()), "uniform must be Float"),
        (lambda: sample(temperature=uniform[:3]), "temperature must hold 5"), (lambda: sample(top_k=p), "top_k must be Int"), (lambda: sample(top_p=uniform.half()), "top_p must be Float"),
        (lambda: sample(min_p=uniform.cpu()), "min_p must be on"), (lambda: sample(u=uniform[:1].expand(5)), "uniform must be contiguous"),
        (lambda: read(bits=8), "rows of 36 do not hold 64"), (lambda: read(bits=2), "row_bits must be 8 or 4"), (lambda: read(dim=63), "even number"), (lambda: read(dim=0), "dim must be in 1"),
        (lambda: read(dtype=torch.float64), "float32, float16 or bfloat16"), (lambda: read(o=offsets.float()), "offsets must be int32 or int64"), (lambda: read(o=offsets[:3]), "block_tables must be int32"),
        (lambda: read(n=-1), "num_tokens must be in"), (lambda: read(starts=offsets), "starts must hold 3"), (lambda: read(kc=c16, vc=c16), "4-bit rows are in a uint8 cache"),
        (lambda: read(kc=c16, vc=c16, bits=8, dtype=torch.float32), "rows come as they are stored"), (lambda: read(vc=u8(4, 2, 16, 40)), "same shape and type"),
        (lambda: append(bits=8), "rows of 36 do not hold 64"), (lambda: append(key=z(3, 2, 63)), "even number"), (lambda: append(kc=u8(4, 2, 16, 37), vc=u8(4, 2, 16, 37)), "4-byte"),
        (lambda: append(vc=u8(4, 1, 16, 36).expand(-1, 2, -1, -1)), "rows of a cache must not overlap"),
        (lambda: attend(bits=8), "rows of 36 do not hold 64"), (lambda: attend(query=z(3, 4, 64, t=torch.float32)), "FP16 or BF16|float16 or bfloat16"), (lambda: attend(kc=c16, vc=c16), "4-bit rows are in a uint8 cache"),
    ]
    for i, (call, word) in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError), match=word):
            call()
            print("not refused:", i)
    # heads of which there are none, and no tokens
    none = rotate(key=k[:, :0])
    assert none[1].shape == (5, 0, 64) and torch.equal(none[0], q)
    assert rotate(query=q[:0], key=k[:0], positions=p[:0])[0].shape == (0, 8, 64)
