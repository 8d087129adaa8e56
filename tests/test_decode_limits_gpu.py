"""The operators of a decoding step at the limits of their arguments and of the number formats they keep."""
import numpy as np
import pytest

import decode_reference as R
from test_decode_finite_gpu import close_and_finite as close
from test_decode_gpu import EDGES, attention_case, make_cache, np64

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


def rows8_sizes(cache, dim):
    """Of every element of 8-bit rows, |scale| |byte - 128| + |bias + 128 scale|: the terms that attention adds up."""
    rows = cache.cpu().numpy()
    pair = np.ascontiguousarray(rows[..., :4]).view(np.float16).astype(np.float64)
    return np.abs(pair[..., :1]) * np.abs(rows[..., 4:4 + dim] - 128.0) + np.abs(pair[..., 1:] + 128 * pair[..., :1])


def attention64(query, values, sizes, tables, lengths, scale, window=0, softcap=0.0):
    """(out, lse, bound of out's error, bound of lse's error) in 64 bits, before the last rounding.

    A score is off by at most (D + 8) 2^-24 of the sum of its terms' sizes and 2^-22 of itself, with a cap by 2^-19 of
    itself: the roundings of scale, ratio and products (10 of 2^-24) and of tanh as a polynomial or as (1 - t) / (1 + t) with
    t <= 1/2 (6 of 2^-23). A weight: the errors of its score and of the maximum, exp2 (2^-22) and the cut to 16 bits (2^-17),
    relatively; the sums' own roundings are within the same 2^-16. Neither bound knows of a cap's size."""
    B, Hq, D = query.shape
    blocks, H, S, _ = values[0].shape
    out, lse = np.zeros((B, Hq, D)), np.full((B, Hq), -np.inf)
    out_off, lse_off = np.zeros((B, Hq, D)), np.zeros((B, Hq))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), tables.shape[1] * S)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = tables[b, t // S]
        if not len(t):
            continue
        for h in range(Hq):
            at = (page, h // (Hq // H), t % S)
            q = query[b, h]
            s = scale * (values[0][at] @ q)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            wrong = (D + 8) * 2.0 ** -24 * abs(scale) * (sizes[0][at] @ np.abs(q)) + (2.0 ** -19 if softcap else 2.0 ** -22) * np.abs(s)
            m = s.max()
            p = np.exp(s - m)
            total = p.sum()
            out[b, h], lse[b, h] = p @ values[1][at] / total, m + np.log(total)
            out_off[b, h] = (2 * wrong.max() + 2.0 ** -15) * (p @ sizes[1][at]) / total
            lse_off[b, h] = wrong.max() + 2.0 ** -20 * (1 + abs(lse[b, h]))
    return out, lse, out_off, lse_off


def check(decode, case, dtype, scale=None, window=0, softcap=0.0):
    query, caches, values, tables, lengths = case
    dim = query.shape[2]
    rows8 = caches[0].dtype == torch.uint8
    sizes = [rows8_sizes(c, dim) if rows8 else np.abs(v) for c, v in zip(caches, values)]
    got, lse = decode.paged_attention(query, *caches, tables, lengths, scale=scale, window=window, softcap=softcap)
    want, want_lse, off, lse_off = attention64(np64(query), values, sizes, tables.cpu().numpy(), lengths.cpu().numpy(),
                                               dim ** -0.5 if scale is None else scale, window, softcap)
    close(got, want, off, dtype)
    close(lse, want_lse, lse_off, torch.float32)


# ---- 8-bit rows -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("hnd", 16), ("nhd", 16), ("hnd", 10)])
@pytest.mark.parametrize("dim", [64, 128, 256, 96])
def test_rows_whose_range_a_single_channel_sets(decode, dim, layout, block, dtype):
    """One element of a row sets its scale, the others are a step or none away from zero: their sums are of a step's size, not of
    the range's, and columns of zeros stay zeros."""
    query, caches, values, tables, lengths = attention_case(decode, dim + block, dim, 4, 2, block, [2, 40, 300, 4099], dtype, True, layout, poison=False)
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    for k, c in enumerate(caches):
        c[..., 4:4 + dim] = torch.randint(127, 130, (*c.shape[:3], dim), device="cuda", generator=g).to(torch.uint8)
        c[..., 4] = torch.where(torch.rand(c.shape[:3], device="cuda", generator=g) < 0.5, 0, 255).to(torch.uint8)
        c[..., 4 + dim // 2: 4 + dim] = 128
        scale = (2.0 / 255 * (0.5 + torch.rand((*c.shape[:3], 1), device="cuda", generator=g))).half()
        c[..., :4] = torch.cat((scale, -128 * scale), -1).view(torch.uint8)
        values[k] = R.rows8_values(c.cpu().numpy(), dim)
    check(decode, (query, caches, values, tables, lengths), dtype)


# ---- caps -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("block", [16, 10])
@pytest.mark.parametrize("softcap", [1e-3, 0.7, 3.0, 30.0, 1e4, 1e6, 1e8, 3e38])
def test_caps_of_every_size(decode, softcap, block, rows8):
    check(decode, attention_case(decode, block, 64, 4, 2, block, [0, 1, 40, 300], torch.float16, rows8), torch.float16, softcap=softcap)


def test_a_cap_that_no_score_meets_is_none(decode):
    q, c, _, t, n = attention_case(decode, 3, 128, 4, 2, 16, [1, 77, 500], torch.bfloat16)
    plain, capped = decode.paged_attention(q, *c, t, n), decode.paged_attention(q, *c, t, n, softcap=1e8)
    # the scores' roundings alone: some 2^-22 of scores below 8
    assert (plain[1] - capped[1]).abs().max() < 2.0 ** -18


@pytest.mark.parametrize("softcap", [1e-36, 1e-40, 1e-44, 1e-50])
def test_caps_below_every_score_leave_equal_weights(decode, softcap):
    """Scores between -softcap and softcap are zero to fp32: every token counts the same, and a score of zero is one of them."""
    query, caches, values, tables, lengths = attention_case(decode, 5, 64, 2, 1, 16, [1, 50, 200], torch.float16)
    query[1] = 0
    out, lse = decode.paged_attention(query, *caches, tables, lengths, softcap=softcap)
    want, want_lse, off, lse_off = attention64(0 * np64(query), [np.nan_to_num(v, posinf=0) for v in values], [np.abs(np.nan_to_num(v, posinf=0)) for v in values],
                                               tables.cpu().numpy(), lengths.cpu().numpy(), 1.0)
    close(out, want, off, torch.float16)
    close(lse, want_lse, lse_off, torch.float32)


# ---- tiles behind tiles -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("hnd", 16), ("hnd", 64), ("nhd", 16), ("hnd", 24)])
@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_tiles_of_a_wave(decode, dim, rows8, layout, block, dtype):
    """64 requests over one context: more steps than the device has workers, so that each wave adds tile behind tile, rows of
    8 bits through its part of LDS."""
    longest, requests = 3000, 64
    query, caches, values, tables, _ = attention_case(decode, dim + block, dim, 4, 4, block, [longest], dtype, rows8, layout)
    g = torch.Generator(device="cuda")
    g.manual_seed(block)
    query = torch.randn((requests, 4, dim), device="cuda", generator=g).to(dtype)
    lengths = longest - torch.arange(requests, device="cuda") * 11
    check(decode, (query, caches, values, tables.expand(requests, -1), lengths), dtype)


# ---- operands that rows share, results over inputs ---------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_and_masks_that_all_rows_share(decode, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rows, vocab = 5, 9001
    one = torch.randn((1, vocab), device="cuda", generator=g).to(dtype)
    words = torch.randint(-(1 << 31), 1 << 31, (1, (vocab + 31) // 32), device="cuda", generator=g).to(torch.int32)
    tokens = torch.randint(0, vocab, (rows * 40,), device="cuda", generator=g)
    offsets = torch.arange(rows + 1, device="cuda") * 40
    penalty = torch.rand(rows, device="cuda", generator=g)
    call = lambda x, m: decode.penalize_logits(x, tokens, offsets, frequency=penalty, mask=m)  # noqa: E731
    want = call(one.repeat(rows, 1), words.repeat(rows, 1))
    assert torch.equal(call(one.expand(rows, -1), words.repeat(rows, 1)), want)
    assert torch.equal(call(one.repeat(rows, 1), words.expand(rows, -1)), want)
    assert torch.equal(call(one.expand(rows, -1), words.expand(rows, -1)), want)


def test_logits_beside_their_result_in_one_tensor(decode):
    """Columns, rows and ends of one tensor that do not meet are fine; logits and results that share elements are refused, but the
    same elements of both."""
    both = torch.randn((4, 2100), device="cuda")
    left, right = both[:, :1000], both[:, 1000:2000]
    penalty = torch.full((4,), 0.5, device="cuda")
    tokens, offsets = torch.arange(40, device="cuda"), torch.arange(5, device="cuda") * 10
    call = lambda x, out=None: decode.penalize_logits(x, tokens, offsets, presence=penalty, out=out)  # noqa: E731
    want = call(left)
    assert torch.equal(call(left, right), want) and torch.equal(right, want)
    rows = torch.randn((8, 2100), device="cuda")  # ends of rows beside the beginnings of others
    want = call(rows[:4, 1000:2000])
    assert torch.equal(call(rows[:4, 1000:2000], rows[2:6, :1000]), want)
    for logits, out in ((left, both[:, 1:1001]), (left, both[:, 999:1999]), (both[:, 500:1500], both[:, 1100:]), (rows[:4, :1000], rows[3:7, :1000]),
                        (left[:1].expand(4, -1), left), (left, right[:1].expand(4, -1)), (left[:1], both[:1, 7:1007])):
        with pytest.raises(RuntimeError, match="overlap"):
            decode.penalize_logits(logits, out=out)


def test_caches_whose_rows_are_one_are_refused(decode):
    new = torch.randn((3, 2, 64), device="cuda").bfloat16()
    slots = torch.arange(3, device="cuda")
    whole = lambda: torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.bfloat16)  # noqa: E731
    shared = [whole()[:1].expand(4, -1, -1, -1), whole()[:, :1].expand(-1, 2, -1, -1), whole()[:, :, :1].expand(-1, -1, 16, -1)]
    for cache in shared:
        with pytest.raises(RuntimeError, match="overlap"):
            decode.kv_cache_append(new, new, cache, whole(), slots)
        with pytest.raises(RuntimeError, match="overlap"):
            decode.kv_cache_append(new, new, whole(), cache, slots)
    same = whole()
    with pytest.raises(RuntimeError, match="overlap"):
        decode.kv_cache_append(new, 2 * new, same, same, slots)
    decode.kv_cache_append(new, new, same, same, slots)  # one row for both
    assert torch.equal(same[0, :, :3], new.transpose(0, 1))
    # keys and values side by side in one tensor are two caches
    both = torch.zeros((4, 2, 2, 16, 64), device="cuda", dtype=torch.bfloat16)
    decode.kv_cache_append(new, 2 * new, both[:, 0], both[:, 1], slots)
    assert torch.equal(both[0, 0, :, :3], new.transpose(0, 1)) and torch.equal(both[0, 1, :, :3], 2 * new.transpose(0, 1))
    # reading rows that are one is nobody's harm
    q = torch.randn((1, 2, 64), device="cuda").bfloat16()
    table, length = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([16], device="cuda")
    kv = torch.randn((1, 1, 16, 64), device="cuda").bfloat16()
    got = decode.paged_attention(q, kv.expand(-1, 2, -1, -1), kv.expand(-1, 2, -1, -1), table, length)
    want = decode.paged_attention(q, kv.repeat(1, 2, 1, 1), kv.repeat(1, 2, 1, 1), table, length)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_as_many_rows_of_logits_as_there_may_be(decode):
    """More than one grid holds: the last rows are those of a second launch, with their own penalties, lists and mask."""
    rows = 1 << 24
    x = torch.arange(rows, device="cuda", dtype=torch.int32).bitwise_and_(1023).half().view(rows, 1)
    x[-3:] = 8
    value = lambda *last: torch.cat((torch.ones(rows - 3, device="cuda"), torch.tensor(last, device="cuda")))  # noqa: E731
    repetition, frequency, presence = value(1.0, 2.0, 4.0), value(1.0, 0.5, 0.25), value(2.0, 0.25, 0.5)
    mask = torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    mask[-3] = 0
    offsets = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    offsets[-3:] = torch.tensor([1, 2, 4], device="cuda", dtype=torch.int32)  # a token of each of the last three rows, two of the last
    prompts = torch.zeros(rows, dtype=torch.int32, device="cuda")
    prompts[-1] = 1  # its first is its prompt's
    zeros = torch.zeros(4, dtype=torch.int32, device="cuda")
    got = decode.penalize_logits(x, zeros, offsets, prompts, repetition=repetition, frequency=frequency, presence=presence,
                                 bias_ids=zeros, bias_values=torch.tensor([1.0, 3.0, 5.0, 7.0], device="cuda"), bias_offsets=offsets, mask=mask)
    want = x.clone()
    want[-3], want[-2], want[-1] = -float("inf"), 8 / 2 - 0.5 - 0.25 + 3, 8 / 4 - 0.25 - 0.5 + 7
    assert torch.equal(got, want)


# ---- numbers that are not finite --------------------------------------------------------------------


@pytest.mark.parametrize("block", [16, 10])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_tokens_that_are_not_finite(decode, dtype, block):
    """A score of -inf weighs nothing, one of +inf or NaN, and a value that is not finite, reach the outputs; a cap makes +inf a number."""
    def run(softcap=0.0):
        return decode.paged_attention(query, *caches, tables, lengths, softcap=softcap)
    query, caches, _, tables, lengths = attention_case(decode, block, 64, 2, 1, block, [200, 90], dtype, poison=False)
    query[:, :, 0] = 1
    page, place = tables[0, 30 // block].long(), 30 % block
    key, value = caches[0][page, 0, place], caches[1][page, 0, place]
    held, kept = key.clone(), value.clone()
    fine = run()
    key[0] = -float("inf")
    without = run()
    assert all(torch.isfinite(x).all() for x in without) and not torch.equal(without[0][0], fine[0][0])
    value[5] = float("nan")
    out, lse = run()
    assert torch.isnan(out[0, :, 5]).all() and torch.isfinite(out[0, :, 6:]).all() and torch.equal(lse, without[1])
    value.copy_(kept)
    key[0] = float("inf")
    out, lse = run()
    assert not torch.isfinite(out[0]).any()
    out, lse = run(softcap=20.0)
    assert torch.isfinite(out).all() and (lse[0] >= 20).all() and (lse[0] < 21).all()  # one score of 20 among others of a few units
    key.copy_(held)
    key[3] = float("nan")
    for got in (run(), run(softcap=20.0)):
        assert torch.isnan(got[0][0]).all() and torch.isnan(got[1][0]).all()
        assert torch.isfinite(got[0][1]).all() and torch.isfinite(got[1][1]).all()  # the other request's tokens are others


# ---- instances of the kernels that other files' shapes do not reach ----------------------------------


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", [7, 16, 24])
@pytest.mark.parametrize("dim", [8, 56, 72, 80, 96, 120, 136, 200, 248])
def test_dims_between_in_pages_of_any_size(decode, dim, block, dtype, rows8):
    check(decode, attention_case(decode, dim + block, dim, 6, 2, block, [0, 1, 40, 133, 300], dtype, rows8), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("nhd", 16), ("padded", 32), ("padded", 10)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_rows_of_8_bits_with_gaps_at_the_edges_of_tiles_and_pages(decode, dim, layout, block, dtype):
    check(decode, attention_case(decode, dim + block, dim, 4, 2, block, EDGES, dtype, True, layout), dtype)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [1, 2, 7, 30, 64, 100, 264, 512, 520])
def test_append_quantizes_rows_of_any_length_from_any_address(decode, dim, dtype, layout, shift):
    from fbgemm_amd import ops
    tokens, heads, block = 37, 3, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    blocks, row = -(-tokens // block) + 1, decode.kv_row_bytes(dim)
    wide = (torch.randn((tokens, 2 * heads, dim + 8), device="cuda", generator=g) - 0.25).to(dtype)
    key, value = wide[:, :heads, shift:shift + dim], wide[:, heads:, shift:shift + dim]
    kc, vc = (make_cache(blocks, heads, block, row, torch.uint8, layout, fill=9) for _ in range(2))
    slots = torch.randperm(blocks * block, device="cuda", generator=g)[:tokens]
    decode.kv_cache_append(key, value, kc, vc, slots)
    for new, cache in ((key, kc), (value, vc)):
        want = torch.full((blocks * block, heads, row), 9, dtype=torch.uint8, device="cuda")
        want[slots, :, : dim + 4] = ops.quantize_rowwise(new.float().reshape(-1, dim), 8, layout=ops.QLAYOUT_TBE).view(tokens, heads, dim + 4)
        assert torch.equal(cache, want.view(blocks, block, heads, row).permute(0, 2, 1, 3))
