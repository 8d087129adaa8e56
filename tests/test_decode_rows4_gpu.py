"""A cache of 4-bit rows: rows written, read back and attended over, against the formulas in 64 bits."""
import numpy as np
import pytest

import decode_reference as R
import decode_tokens_reference as T
from test_decode_finite_gpu import close_and_finite as close
from test_decode_gpu import EDGES, make_cache, np64

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


# ---- rows written -----------------------------------------------------------------------------------


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,block", [(1, 1, 2, 1), (5, 3, 8, 4), (64, 8, 128, 16), (33, 2, 80, 5), (300, 5, 256, 24), (37, 3, 30, 5), (3, 1, 1000, 64), (9, 2, 520, 7)])
def test_append_quantizes_rows_as_the_quantizer_does(decode, tokens, heads, dim, block, dtype, layout, shift):
    from fbgemm_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + dim)
    blocks, row = -(-tokens // block) + 3, decode.kv_row_bytes(dim, 4)
    fused = (torch.randn((tokens, 2 * heads, dim + 8), device="cuda", generator=g) + 0.25).to(dtype)
    fused[0, 0] = 3.0  # a constant row
    key, value = fused[:, :heads, shift:shift + dim], fused[:, heads:, shift:shift + dim]
    kc, vc = (make_cache(blocks, heads, block, row, torch.uint8, layout, fill=9) for _ in range(2))
    slots = torch.randperm(blocks * block, device="cuda", generator=g)[:tokens]
    slots[tokens // 2] = -1
    decode.kv_cache_append(key, value, kc, vc, slots, row_bits=4)
    keep = slots >= 0
    for new, cache in ((key, kc), (value, vc)):
        want = torch.full((blocks * block, heads, row), 9, dtype=torch.uint8, device="cuda")
        rows = ops.quantize_rowwise(new.float().reshape(-1, dim), 4, layout=ops.QLAYOUT_TBE)
        want[slots[keep], :, : dim // 2 + 4] = rows.view(tokens, heads, dim // 2 + 4)[keep]
        assert torch.equal(cache, want.view(blocks, block, heads, row).permute(0, 2, 1, 3))


def test_append_of_numbers_that_the_format_does_not_hold(decode):
    """Elements beyond fp16's largest number count as that one, NaN as 0; rows whose steps are below fp16's smallest."""
    from fbgemm_amd import ops
    x = torch.randn((8, 1, 64), device="cuda")
    x[0, 0, 5], x[1, 0, 6], x[2, 0, 7], x[3, 0, 8], x[4] = float("inf"), -float("inf"), float("nan"), 1e30, float("nan")
    x[5], x[6] = 1e-7 * x[5], 3e-6 * x[6].abs()
    kc, vc = (make_cache(1, 1, 8, 36, torch.uint8, "hnd", fill=0) for _ in range(2))
    for dtype in (torch.float32, torch.bfloat16):
        new = x.to(dtype)
        decode.kv_cache_append(new, new, kc, vc, torch.arange(8, device="cuda"), row_bits=4)
        want = ops.quantize_rowwise(new.float().nan_to_num(nan=0.0).clamp(-65504, 65504).reshape(8, 64), 4, layout=ops.QLAYOUT_TBE)
        assert torch.equal(kc[0, 0], want) and torch.equal(vc, kc)


def test_append_reports_slots_outside_the_cache(decode):
    from fbgemm_amd import ops
    new = torch.randn((9, 2, 64), device="cuda").bfloat16()
    kc, vc = (make_cache(2, 2, 4, 36, torch.uint8, "hnd", fill=1) for _ in range(2))
    st = ops.Status()
    for slots, want in (([0, 1, 2, -1, 3, 4, 5, -1, 6], (0, -1)), ([0, 1, 8, 2, -2, 3, 4, 5, 1 << 40], (1, 2))):
        st.clear()
        decode.kv_cache_append(new, new, kc, vc, torch.tensor(slots, device="cuda"), status=st, row_bits=4)
        assert st.read() == want
    assert (kc[1, :, 3] == 1).all()  # the slot that nobody had


# ---- rows read back ---------------------------------------------------------------------------------


def read_case(decode, seed, lengths, starts, heads, dim, block, store, layout):
    """(caches, their values in fp32 [blocks, heads, block, dim], tables, offsets, starts)"""
    rng = np.random.default_rng(seed)
    spans = [n + s for n, s in zip(lengths, starts or [0] * len(lengths))]
    used = [-(-n // block) for n in spans]
    blocks, width = sum(used) + 2, max(used + [1])
    pages = rng.permutation(blocks).astype(np.int32)
    tables = np.full((len(lengths), width), 1 << 30, np.int32)
    at = 0
    for r, n in enumerate(used):
        tables[r, :n] = pages[at:at + n]
        at += n
    caches, values = [], []
    for _ in range(2):
        if store in (4, 8):
            c = make_cache(blocks, heads, block, decode.kv_row_bytes(dim, store), torch.uint8, layout)
            c.copy_(torch.from_numpy(rng.integers(0, 256, c.shape, dtype=np.uint8)))
            pair = torch.from_numpy(rng.uniform(-2, 2, (*c.shape[:3], 2))).half().cuda()
            c[..., :4] = pair.view(torch.uint8)
            host = c.cpu().numpy()
            codes = T.codes4(host, dim) if store == 4 else host[..., 4:4 + dim].astype(np.float64)
            pair = pair.cpu().numpy().astype(np.float64)
            values.append((codes * pair[..., :1] + pair[..., 1:]).astype(np.float32))
        else:
            c = make_cache(blocks, heads, block, dim, store, layout)
            c.copy_(torch.from_numpy(rng.standard_normal(c.shape)))
            values.append(c.cpu().float().numpy())
        caches.append(c)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    return caches, values, tables, offsets, starts


def check_read(decode, case, store, dtype, index, num_tokens, dim):
    from fbgemm_amd import ops
    caches, values, tables, offsets, starts = case
    st = ops.Status()
    cu = lambda a: torch.from_numpy(np.asarray(a, index)).cuda()  # noqa: E731
    got = decode.kv_cache_read(*caches, torch.from_numpy(tables).cuda(), cu(offsets), num_tokens, dim, dtype, None if starts is None else cu(starts), status=st,
                               row_bits=store if store in (4, 8) else 8)
    for g, v in zip(got, values):
        want, bad = T.read(v, tables, offsets, starts, num_tokens)
        assert g.dtype == (dtype or (torch.float32 if store in (4, 8) else store)) and g.shape == want.shape
        assert torch.equal(g.cpu(), torch.from_numpy(want).to(g.dtype))
    assert st.read() == ((1, min(bad)) if bad else (0, -1))
    return bad


STORES = [(4, None), (4, torch.float16), (4, torch.bfloat16), (8, torch.float32), (8, torch.bfloat16), (torch.float32, None), (torch.float16, torch.float16), (torch.bfloat16, None)]


@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("store,dtype", STORES)
@pytest.mark.parametrize("heads,dim,block", [(1, 2, 1), (3, 8, 7), (8, 128, 16), (2, 80, 24), (5, 30, 16), (1, 1000, 3), (2, 256, 64)])
def test_read(decode, heads, dim, block, store, dtype, layout):
    lengths = [0, 1, 33, 0, 0, 70, 5, 0]
    check_read(decode, read_case(decode, dim, lengths, None, heads, dim, block, store, layout), store, dtype, np.int32, sum(lengths), dim)
    starts = [3, 0, 17, 0, 9, 70, 1000, 5]
    check_read(decode, read_case(decode, dim + 1, lengths, starts, heads, dim, block, store, layout), store, dtype, np.int64, sum(lengths) + 9, dim)


@pytest.mark.parametrize("store", [4, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 2047, 2049, 16383, 16390, 40000])
def test_read_of_many_tokens(decode, tokens, store):
    rng = np.random.default_rng(tokens)
    cuts = np.sort(rng.integers(0, tokens + 1, 40))
    lengths = np.diff(np.concatenate([[0], cuts, [tokens]])).tolist()
    check_read(decode, read_case(decode, 1, lengths, None, 2, 16, 16, store, "hnd"), store, None, np.int32, tokens, 16)


@pytest.mark.parametrize("store,dtype,tokens", [(4, torch.float32, 16_500), (4, torch.bfloat16, 33_001), (8, torch.float16, 33_001), (torch.bfloat16, None, 33_001)])
def test_read_past_the_caches_gives_the_same_bits(decode, store, dtype, tokens):
    """Results of more than 128 MB, and the same tokens in parts."""
    blocks = -(-tokens // 16)
    caches = [torch.randn((blocks, 8, 16, 128), device="cuda").bfloat16() for _ in "kv"]
    bits = store if store in (4, 8) else 8
    if store in (4, 8):
        for i, c in enumerate(caches):
            caches[i] = torch.randint(0, 256, (*c.shape[:3], decode.kv_row_bytes(128, store)), dtype=torch.uint8, device="cuda")
            caches[i][..., :4] = torch.randn((*c.shape[:3], 2), device="cuda").half().view(torch.uint8)
    tables = torch.randperm(blocks, device="cuda").int()[None]
    at = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    got = decode.kv_cache_read(*caches, tables, at(0, tokens), tokens, 128, dtype, row_bits=bits)
    for first in range(0, tokens, 1999):
        n = min(1999, tokens - first)
        want = decode.kv_cache_read(*caches, tables, at(0, n), n, 128, dtype, at(first), row_bits=bits)
        assert all(torch.equal(x[first:first + n], y) for x, y in zip(got, want))


@pytest.mark.parametrize("store", [4, 8, torch.float16])
def test_read_of_tokens_without_a_page(decode, store):
    lengths, starts = [20, 40, 5], [0, 8, 0]
    for change in (lambda t, s: t.__setitem__((1, 1), -1), lambda t, s: t.__setitem__((0, 0), 1 << 29), lambda t, s: s.__setitem__(2, -3), lambda t, s: s.__setitem__(1, 1 << 40),
                   lambda t, s: s.__setitem__(0, 10_000)):
        case = read_case(decode, 3, lengths, list(starts), 2, 64, 16, store, "hnd")
        change(case[2], case[4])
        assert check_read(decode, case, store, None, np.int64, 70, 64)
    caches, _, tables, offsets, _ = read_case(decode, 3, lengths, starts, 2, 64, 16, store, "hnd")
    t, o = torch.from_numpy(tables).cuda(), torch.from_numpy(offsets).cuda()
    bits = store if store in (4, 8) else 8
    for args in ((*[c[:0] for c in caches], t, o), (*caches, t[:, :0], o), (*caches, t[:0], o[:1])):
        got = decode.kv_cache_read(*args, 65, 64, row_bits=bits)
        assert (got[0] == 0).all() and (got[1] == 0).all() and got[0].shape == (65, 2, 64)
    assert decode.kv_cache_read(*caches, t, o, 0, 64, row_bits=bits)[0].shape == (0, 2, 64)
    # offsets that do not ascend give something, of rows that are there
    got = decode.kv_cache_read(*caches, t, torch.tensor([40, 3, 60, 20], device="cuda"), 65, 64, row_bits=bits)
    assert got[0].shape == (65, 2, 64)


def test_what_is_written_is_read_back(decode):
    from fbgemm_amd import ops
    x = torch.randn((77, 4, 96), device="cuda").bfloat16()
    for bits in (4, 8):
        kc, vc = (torch.zeros((9, 4, 16, decode.kv_row_bytes(96, bits)), dtype=torch.uint8, device="cuda") for _ in range(2))
        tables = torch.randperm(9, device="cuda").int().view(1, 9)
        p = torch.arange(77, device="cuda")
        decode.kv_cache_append(x, 2 * x, kc, vc, tables[0, p // 16].long() * 16 + p % 16, row_bits=bits)
        key, value = decode.kv_cache_read(kc, vc, tables, torch.tensor([0, 77], device="cuda"), 77, 96, row_bits=bits)
        for new, got in ((x, key), (2 * x, value)):
            rows = ops.quantize_rowwise(new.float().reshape(-1, 96), bits, layout=ops.QLAYOUT_TBE)
            assert torch.equal(got.view(-1, 96), ops.dequantize_rowwise(rows, 96, bits, layout=ops.QLAYOUT_TBE))


def test_read_beyond_32_bit_offsets(decode):
    """The last pages of a cache of 9 GiB."""
    blocks = 9 * (1 << 30) // (8 * 64 * 68)
    c = torch.zeros((blocks, 8, 64, 68), dtype=torch.uint8, device="cuda")
    c[blocks - 1] = torch.randint(0, 100, (8, 64, 68), device="cuda", dtype=torch.uint8)
    key, value = decode.kv_cache_read(c, c, torch.tensor([[3, blocks - 1]], dtype=torch.int32, device="cuda"), torch.tensor([0, 128], device="cuda"), 128, 128, row_bits=4)
    want = torch.from_numpy(T.rows4_values(c[blocks - 1].cpu().numpy(), 128)).float().transpose(0, 1)
    assert torch.equal(key[64:].cpu(), want) and torch.equal(value, key) and (key[:64] == 0).all()


# ---- attention --------------------------------------------------------------------------------------


def attention4(query, caches, tables, lengths, scale, window=0, softcap=0.0):
    """(out, lse, bound of out's error, bound of lse's error) in 64 bits, before the last rounding.

    Scores are a (q . n) + b sum(q): (D + 8) 2^-24 of the sum of these terms' sizes (a n and b by |q|), and 2^-22 of themselves, with a cap
    2^-19. A weight: its score's and the maximum's errors, exp2 (2^-22) and the cut to 16 bits (2^-17), relatively, of p |a| |n - 8| and p |b + 8 a|: codes
    and their eights have the same cut weights. Both are sums of codes up to 15, of as many additions as there are tiles of a wave and a
    few: 2^-24 of p |a| 15 each."""
    B, Hq, D = query.shape
    blocks, H, S, _ = caches[0].shape
    out, lse = np.zeros((B, Hq, D)), np.full((B, Hq), -np.inf)
    out_off, lse_off = np.zeros((B, Hq, D)), np.zeros((B, Hq))
    pairs = [np.ascontiguousarray(c[..., :4]).view(np.float16).astype(np.float64) for c in caches]
    for r in range(B):
        n = min(max(int(lengths[r]), 0), tables.shape[1] * S)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = tables[r, t // S]
        t, page = t[(page >= 0) & (page < blocks)], page[(page >= 0) & (page < blocks)]
        if not len(t):
            continue
        for h in range(Hq):
            at = (page, h // (Hq // H), t % S)
            q = query[r, h]
            k, v = (T.codes4(c[at], D) for c in caches)
            (ka, kb), (va, vb) = ((p[at][:, :1], p[at][:, 1:]) for p in pairs)
            s = scale * ((ka * k + kb) @ q)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            wrong = (D + 8) * 2.0 ** -24 * abs(scale) * ((np.abs(ka) * k + np.abs(kb)) @ np.abs(q)) + (2.0 ** -19 if softcap else 2.0 ** -22) * np.abs(s)
            m = s.max()
            p = np.exp(s - m)
            total = p.sum()
            out[r, h], lse[r, h] = p @ (va * v + vb) / total, m + np.log(total)
            sizes = np.abs(va) * np.abs(v - 8) + np.abs(vb + 8 * va)
            out_off[r, h] = ((2 * wrong.max() + 2.0 ** -15) * (p @ sizes) + (len(t) / 64 + 12) * 2.0 ** -24 * 15 * (p @ np.abs(va))) / total
            lse_off[r, h] = wrong.max() + 2.0 ** -20 * (1 + abs(lse[r, h]))
    return out, lse, out_off, lse_off


def attention_case(decode, seed, dim, heads, kv_heads, block, lengths, dtype, layout="hnd", index=torch.int32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B = len(lengths)
    used = [-(-max(n, 0) // block) for n in lengths]
    blocks, width = sum(used) + 2, max(max(used), 1)
    pages = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((B, width), 1 << 30, dtype=torch.int32, device="cuda")
    written = torch.zeros((blocks, block), dtype=torch.bool, device="cuda")
    at = 0
    for b, n in enumerate(lengths):
        tables[b, :used[b]] = pages[at:at + used[b]]
        for j in range(used[b]):
            written[pages[at + j].long(), : min(block, n - j * block)] = True
        at += used[b]
    query = torch.randn((B, heads, dim), device="cuda", generator=g).to(dtype)
    caches = []
    for _ in range(2):
        c = make_cache(blocks, kv_heads, block, decode.kv_row_bytes(dim, 4), torch.uint8, layout)
        c.copy_(torch.randint(0, 256, c.shape, device="cuda", generator=g, dtype=torch.uint8))
        scale = 4.0 / 15 * (0.5 + torch.rand((*c.shape[:3], 1), device="cuda", generator=g))
        c[..., :4] = torch.cat((scale, scale * -15 * torch.rand(scale.shape, device="cuda", generator=g)), -1).half().view(torch.uint8)
        c.masked_fill_(~written[:, None, :, None], 255)  # scales and biases of rows without a token: NaN
        caches.append(c)
    return query, caches, tables, torch.tensor(lengths, device="cuda", dtype=index)


def check(decode, case, dtype, scale=None, window=0, softcap=0.0):
    query, caches, tables, lengths = case
    call = lambda: decode.paged_attention(query, *caches, tables, lengths, scale=scale, window=window, softcap=softcap, row_bits=4)  # noqa: E731
    got, lse = call()
    assert got.dtype == dtype and got.shape == query.shape and lse.dtype == torch.float32
    s = query.shape[2] ** -0.5 if scale is None else scale
    want, want_lse, off, lse_off = attention4(np64(query), [c.cpu().numpy() for c in caches], tables.cpu().numpy(), lengths.cpu().numpy(), s, window, softcap)
    close(got, want, off, dtype)
    close(lse, want_lse, lse_off, torch.float32)
    again = call()
    assert torch.equal(again[0], got) and torch.equal(again[1], lse)  # the same bits every time


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("hnd", 1), ("hnd", 7), ("hnd", 16), ("hnd", 24), ("hnd", 48), ("hnd", 64), ("nhd", 16), ("padded", 32), ("padded", 10)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_at_the_edges_of_tiles_and_pages(decode, dim, layout, block, dtype):
    check(decode, attention_case(decode, dim + block, dim, 4, 2, block, EDGES, dtype, layout), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", [7, 16, 24])
@pytest.mark.parametrize("dim", [8, 24, 40, 56, 72, 80, 96, 120, 136, 192, 200, 248])
def test_attention_of_dims_between(decode, dim, block, dtype):
    check(decode, attention_case(decode, dim, dim, 6, 2, block, [0, 1, 40, 133, 300], dtype), dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (6, 2), (7, 1), (15, 1), (16, 1), (17, 1), (32, 2), (66, 2), (40, 1)])
def test_attention_of_shared_heads(decode, heads, kv_heads):
    check(decode, attention_case(decode, heads, 64, heads, kv_heads, 16, [3, 0, 200, 65], torch.float16), torch.float16)
    check(decode, attention_case(decode, heads, 128, heads, kv_heads, 16, [3, 0, 200, 65], torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize("block", [16, 10])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0.0, None), (17, 0.0, 0.3), (128, 5.0, None), (1000, 30.0, 0.5), (0, 2.0, -0.2), (130, 0.0, 0.0), (0, 1e-3, None), (0, 1e8, None)])
def test_attention_with_a_window_a_cap_and_a_scale(decode, window, softcap, scale, block):
    case = attention_case(decode, window, 128, 4, 2, block, [0, 1, 16, 129, 130, 131, 500], torch.float16, index=torch.int64)
    check(decode, case, torch.float16, scale, window, softcap)


@pytest.mark.parametrize("block", [16, 12])
def test_attention_split_over_workers(decode, block):
    check(decode, attention_case(decode, 5, 64, 8, 2, block, [9000, 0, 1, 20011, 0, 128, 4097], torch.bfloat16), torch.bfloat16)
    check(decode, attention_case(decode, 6, 128, 2, 1, block, [70003], torch.float16), torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("hnd", 16), ("nhd", 16), ("hnd", 24)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_tiles_of_a_wave(decode, dim, layout, block, dtype):
    """64 requests over one context: more steps than the device has workers, so that each wave adds tile behind tile."""
    longest, requests = 3000, 64
    query, caches, tables, _ = attention_case(decode, dim + block, dim, 4, 4, block, [longest], dtype, layout)
    g = torch.Generator(device="cuda")
    g.manual_seed(block)
    query = torch.randn((requests, 4, dim), device="cuda", generator=g).to(dtype)
    check(decode, (query, caches, tables.expand(requests, -1), longest - torch.arange(requests, device="cuda") * 11), dtype)


@pytest.mark.parametrize("block", [16, 10])
def test_attention_leaves_out_blocks_that_are_not_there(decode, block):
    query, caches, tables, lengths = attention_case(decode, 8, 128, 4, 2, block, [100, 64, 31, 16], torch.float16)
    tables[0, 1], tables[0, 3], tables[1], tables[2, 0] = -1, 1 << 29, -1, caches[0].shape[0]
    check(decode, (query, caches, tables, lengths), torch.float16)
    # lengths below zero and beyond the table, of pages that are full (rows without a token are NaN, and these lengths would have them)
    query, caches, tables, _ = attention_case(decode, 9, 128, 4, 2, block, [8 * block, 3 * block, 8 * block, block], torch.float16)
    check(decode, (query, caches, tables, torch.tensor([-4, 1000, 1 << 40, 3], device="cuda")), torch.float16)


@pytest.mark.parametrize("power", [-130, -100, -20, 0, 14, 60, 110])
def test_queries_of_every_size(decode, power):
    """bf16 queries from subnormal numbers to 2^112, beside elements 2^-30 as large and zeros: scores near 1 by the scale."""
    query, caches, tables, lengths = attention_case(decode, 3, 128, 4, 2, 16, [1, 33, 200], torch.bfloat16)
    query = query * 2.0 ** power if power > -120 else (query.double() * 2.0 ** power).float().bfloat16()
    query[:, :, ::3] *= 2.0 ** -30 if power > -90 else 1
    query[1, 0] = 0
    check(decode, (query.contiguous(), caches, tables, lengths), torch.bfloat16, scale=float(np.float32(min(2.0 ** (-power - 4), 3e38))))


def test_fp16_queries_of_every_size(decode):
    for power in (-24, -14, 0, 12):
        query, caches, tables, lengths = attention_case(decode, 3, 128, 4, 2, 16, [1, 33, 200], torch.float16)
        check(decode, ((query.float() * 2.0 ** power).half(), caches, tables, lengths), torch.float16, scale=2.0 ** (-power - 4))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,block", [("hnd", 16), ("nhd", 16), ("hnd", 10)])
@pytest.mark.parametrize("dim", [64, 128, 256, 96])
def test_columns_of_zeros_stay_zeros(decode, dim, layout, block, dtype):
    """Code 8 of rows that lie about zero stands for zero: codes' and eights' sums are the same there, bit by bit, at even and odd columns."""
    query, caches, tables, lengths = attention_case(decode, dim + block, dim, 4, 2, block, [2, 40, 300, 4099], dtype, layout)
    for c in caches:
        pair = c[..., :4].clone().view(torch.float16)
        written = ~torch.isnan(pair[..., :1].float())
        pair[..., 1:] = torch.where(written, -8 * pair[..., :1], pair[..., 1:])
        c[..., :4] = pair.view(torch.uint8)
    caches[1][..., 4 + dim // 4: 4 + dim // 2] = 0x88
    out, _ = decode.paged_attention(query, *caches, tables, lengths, row_bits=4)
    assert (out[..., dim // 2:] == 0).all()
    check(decode, (query, caches, tables, lengths), dtype)


@pytest.mark.parametrize("power", [-20, -10, 10])
def test_scales_of_every_size(decode, power):
    """fp16 scales down to subnormal ones, and large ones: weights go to the products times the scale."""
    query, caches, tables, lengths = attention_case(decode, 4, 128, 4, 2, 16, [1, 33, 200], torch.bfloat16)
    for c in caches:
        pair = c[..., :4].clone().view(torch.float16)
        c[..., :4] = (pair.float() * 2.0 ** power).half().view(torch.uint8)
    check(decode, (query, caches, tables, lengths), torch.bfloat16, scale=2.0 ** -power / 8)


def test_attention_of_tokens_that_are_not_finite(decode):
    """A token whose scale or bias is not finite reaches its queries' outputs, and no other request's."""
    for dtype in (torch.float16, torch.bfloat16):
        query, caches, tables, lengths = attention_case(decode, 16, 64, 2, 1, 16, [200, 90], dtype)
        call = lambda: decode.paged_attention(query, *caches, tables, lengths, row_bits=4)  # noqa: E731
        fine = call()
        page = tables[0, 1].long()
        for k in range(2):
            held = caches[k][page].clone()
            caches[k][page, 0, 14, :4] = 255
            out, lse = call()
            assert torch.isnan(out[0]).all() and torch.equal(out[1], fine[0][1]) and torch.isnan(lse[0]).all() == (k == 0) and torch.equal(lse[1], fine[1][1])
            caches[k][page] = held
        query[0, 0, 3] = float("inf")
        out, lse = call()
        assert not torch.isfinite(out[0, 0]).any() and torch.equal(out[0, 1], fine[0][0, 1]) and torch.equal(out[1], fine[0][1])


def test_attention_of_one_word_rows_over_a_large_cache(decode):
    """Pages beyond 4 GiB."""
    blocks, block = 17000, 64
    kc, vc = (torch.zeros((blocks, 8, block, 68), dtype=torch.uint8, device="cuda") for _ in range(2))
    pages = [blocks - 1, 3, blocks // 2 + 1, 16384]
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    query = torch.randn((1, 16, 128), device="cuda", generator=g).bfloat16()
    rows = torch.randn((2, 200, 8, 128), device="cuda", generator=g).bfloat16()
    slots = torch.tensor([pages[t // block] * block + t % block for t in range(200)], device="cuda")
    decode.kv_cache_append(rows[0], rows[1], kc, vc, slots, row_bits=4)
    got, lse = decode.paged_attention(query, kc, vc, torch.tensor([pages], dtype=torch.int32, device="cuda"), torch.tensor([200], device="cuda"), row_bits=4)
    small = [c[torch.tensor(pages, device="cuda")].cpu().numpy() for c in (kc, vc)]
    want, want_lse, off, lse_off = attention4(np64(query), small, np.arange(4)[None], np.array([200]), 128 ** -0.5)
    close(got, want, off, torch.bfloat16)
    close(lse, want_lse, lse_off, torch.float32)


# ---- several calls ----------------------------------------------------------------------------------


def test_attention_on_two_streams_at_once_and_call_behind_call(decode):
    cases = [attention_case(decode, 20 + k, 128, 2, 1, 16, lengths, torch.bfloat16) for k, lengths in enumerate(([30011, 5, 4099], [20011, 300, 5]))]
    call = lambda c: decode.paged_attention(c[0], *c[1], c[2], c[3], row_bits=4)  # noqa: E731
    want = []
    for c in cases:
        want.append(call(c))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((k, call(cases[k])))
    torch.cuda.synchronize()
    got += [(k, call(cases[k])) for k in (0, 1, 0, 0, 1, 1, 0, 1)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k, pair in got for a, b in zip(pair, want[k]))


def test_refusals(decode):
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda")  # noqa: E731
    kv, c4, slots = torch.zeros((3, 2, 64), device="cuda").half(), u8(4, 2, 16, 36), torch.arange(3, device="cuda")
    q, tables, lengths, offsets = torch.zeros((3, 4, 64), device="cuda").half(), torch.zeros((3, 2), device="cuda").int(), torch.ones(3, device="cuda").int(), torch.arange(4, device="cuda")
    append = lambda key=kv, value=kv, kc=c4, vc=c4, row_bits=4: decode.kv_cache_append(key, value, kc, vc, slots, row_bits=row_bits)  # noqa: E731
    attend = lambda query=q, kc=c4, vc=c4, row_bits=4: decode.paged_attention(query, kc, vc, tables, lengths, row_bits=row_bits)  # noqa: E731
    read = lambda kc=c4, vc=c4, t=tables, o=offsets, n=3, dim=64, dtype=None, starts=None, row_bits=4: decode.kv_cache_read(kc, vc, t, o, n, dim, dtype, starts, row_bits=row_bits)  # noqa: E731
    c16 = torch.zeros((4, 2, 16, 64), device="cuda").half()
    refused = [
        lambda: append(row_bits=8), lambda: append(row_bits=2), lambda: append(kc=u8(4, 2, 16, 32), vc=u8(4, 2, 16, 32)), lambda: append(kc=c16, vc=c16),
        lambda: append(key=kv[..., :63], value=kv[..., :63]), lambda: append(kc=u8(4, 2, 16, 37), vc=u8(4, 2, 16, 37)), lambda: append(value=2 * kv),
        lambda: append(kc=u8(4, 1, 16, 36).expand(-1, 2, -1, -1), vc=u8(4, 2, 16, 36)),
        lambda: attend(row_bits=8), lambda: attend(row_bits=16), lambda: attend(kc=c16, vc=c16), lambda: attend(query=q.float()), lambda: attend(query=q[..., :60]),
        lambda: attend(kc=u8(4, 2, 16, 37), vc=u8(4, 2, 16, 37)), lambda: attend(kc=u8(4, 3, 16, 36), vc=u8(4, 3, 16, 36)),
        lambda: read(row_bits=8), lambda: read(dim=63), lambda: read(dim=0), lambda: read(dtype=torch.float64), lambda: read(dtype=torch.uint8), lambda: read(o=offsets.float()),
        lambda: read(o=offsets[:3]), lambda: read(o=offsets[:0], t=tables[:0]), lambda: read(t=tables.long()), lambda: read(t=tables[:2]), lambda: read(n=-1), lambda: read(starts=offsets),
        lambda: read(starts=lengths), lambda: read(o=offsets.cpu()), lambda: read(kc=c16, vc=c16, row_bits=8, dtype=torch.float32), lambda: read(vc=u8(4, 2, 16, 40)),
        lambda: read(kc=c16, vc=c16),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError, TypeError, NotImplementedError)):
            call()
            print("not refused:", i)
    append(vc=u8(4, 2, 16, 36)), attend(), read(kc=c16, vc=c16, row_bits=8)
    torch.cuda.synchronize()
