"""The operators of a decoding step (fbgemm_amd/decode.py) against their formulas in 64 bits, at the sizes, masks, strides and
contents where they can go wrong, and what they refuse."""
import numpy as np
import pytest

import decode_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # of a number rounded to the type, relatively
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


def cu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def np64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, off, dtype):
    """`got` within `off` of `want`, and one rounding to its type; infinities and zeros where `want` has them."""
    got = np64(got)
    fine = np.isfinite(want)
    assert (got[~fine] == want[~fine]).all()
    got, want, off = got[fine], want[fine], np.broadcast_to(off, fine.shape)[fine]
    bad = np.abs(got - want) > off + HALF_ULP[dtype] * (np.abs(want) + off) + SMALLEST[dtype]
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], off[bad][:4])


# ---- block tables -----------------------------------------------------------------------------------


def tables_case(rng, requests, block, width, most_held, most_new, spare=8):
    held = rng.integers(0, most_held + 1, requests)
    new = rng.integers(0, most_new + 1, requests)
    old, need = -(-held // block), -(-(held + new) // block)
    pages = rng.permutation(int(need.sum()) + spare).astype(np.int32)
    tables = np.full((requests, width), -1, np.int32)
    at = 0
    for r in range(requests):
        tables[r, :old[r]] = pages[at:at + old[r]]
        at += old[r]
    return held, new, tables, pages, at


def run_tables(decode, held, new, tables, free, start, block, num_tokens, index, again=True):
    from fbgemm_amd import ops
    t = tables if torch.is_tensor(tables) else cu(tables)
    st = ops.Status()
    args = (cu(held.astype(index)), cu(new.astype(index)), t, cu(free), cu(np.array([start], np.int32)), block, num_tokens)
    want = R.block_tables(held, new, t.cpu().numpy(), free, start, block, num_tokens)
    for _ in range(2 if again else 1):  # the same call gives the same again
        got = decode.kv_block_tables(*args, status=st)
        assert (t.cpu().numpy() == want[0]).all()
        assert (got.slots.cpu().numpy() == want[1]).all()
        assert (got.positions.cpu().numpy() == want[2]).all()
        assert (got.offsets.cpu().numpy() == want[3]).all() and got.offsets.dtype == torch.int32
        assert (got.lengths.cpu().numpy() == want[4]).all() and got.lengths.dtype == args[0].dtype
        assert got.free_start.item() == want[5]
    assert st.read()[0] == want[6]
    return got


@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("requests,block,most_held,most_new", [
    (1, 16, 0, 0), (1, 1, 5, 9), (3, 16, 40, 1), (64, 16, 300, 1), (65, 24, 300, 70), (7, 7, 100, 3000), (200, 128, 1000, 2),
    (5000, 16, 60, 2), (9000, 3, 5, 5)])
def test_block_tables(decode, requests, block, most_held, most_new, index):
    rng = np.random.default_rng(requests + block)
    width = -(-(most_held + most_new) // block) + 1
    held, new, tables, free, start = tables_case(rng, requests, block, width, most_held, most_new)
    run_tables(decode, held, new, tables, free, start, block, int(new.sum()), index)


def test_block_tables_of_no_requests_and_of_none_with_tokens(decode):
    none = np.zeros(0, np.int64)
    run_tables(decode, none, none, np.zeros((0, 4), np.int32), np.arange(3, dtype=np.int32), 1, 16, 0, np.int64)
    run_tables(decode, none, none, np.zeros((0, 4), np.int32), np.arange(3, dtype=np.int32), 1, 16, 5, np.int64)
    run_tables(decode, np.array([5, 0, 17]), np.zeros(3, np.int64), np.arange(12, dtype=np.int32).reshape(3, 4), np.zeros(0, np.int32), 0, 8, 0, np.int32)


def test_block_tables_padded_and_cut_lists_of_tokens(decode):
    rng = np.random.default_rng(1)
    held, new, tables, free, start = tables_case(rng, 40, 16, 12, 100, 30)
    for num in (int(new.sum()) + 37, int(new.sum()) - 11):
        run_tables(decode, held, new, tables, free, start, 16, num, np.int32)


def test_block_tables_with_too_few_blocks_too_narrow_a_table_and_negative_lengths(decode):
    rng = np.random.default_rng(2)
    held, new, tables, free, start = tables_case(rng, 50, 16, 12, 100, 60)
    run_tables(decode, held, new, tables, free[: start + 20], start, 16, int(new.sum()), np.int64)   # the list ends early
    run_tables(decode, held, new, tables, free, -3, 16, int(new.sum()), np.int64)                      # a place before it
    run_tables(decode, held, new, tables[:, :5], free, start, 16, int(new.sum()), np.int64)            # some tokens have no column
    held, new = held.copy(), new.copy()
    held[3], new[7], new[9] = -5, -1, 0
    run_tables(decode, held, new, tables, free, start, 16, int(np.maximum(new, 0).sum()), np.int32)
    # entries that hold no block give their tokens no slot
    tables = tables.copy()
    tables[:, 0] = -1
    run_tables(decode, np.full(50, 3), np.full(50, 2), tables, free, start, 16, 100, np.int32)


def test_block_tables_of_a_wider_tensor_leave_the_rest_alone(decode):
    rng = np.random.default_rng(3)
    held, new, tables, free, start = tables_case(rng, 30, 16, 9, 80, 40)
    whole = torch.full((30, 20), -7, dtype=torch.int32, device="cuda")
    whole[:, 4:13] = cu(tables)
    run_tables(decode, held, new, whole[:, 4:13], free, start, 16, int(new.sum()), np.int64)
    assert (whole[:, :4] == -7).all() and (whole[:, 13:] == -7).all()


# ---- cache rows -------------------------------------------------------------------------------------


def make_cache(blocks, heads, block, row, dtype, layout, fill=None):
    """A cache [blocks, heads, block, row] of one of the layouts: heads outside tokens ("hnd"), inside them ("nhd"), or padded."""
    shape = (blocks, heads, block, row)
    if layout == "hnd":
        c = torch.empty(shape, dtype=dtype, device="cuda")
    elif layout == "nhd":
        c = torch.empty((blocks, block, heads, row), dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    else:
        pad = 16 if dtype == torch.uint8 else 8
        c = torch.empty((blocks, heads + 1, block + 3, row + pad), dtype=dtype, device="cuda")[:, :heads, :block, :row]
    if fill is not None:
        c.fill_(fill)
    return c


@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,block", [(1, 1, 1, 1), (5, 3, 7, 4), (64, 8, 128, 16), (33, 2, 10, 5), (700, 5, 96, 24), (3, 1, 300, 64)])
def test_append_copies_rows(decode, tokens, heads, dim, block, dtype, layout):
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    blocks = -(-tokens // block) + 3
    fused = torch.randn((tokens, 4 * heads, dim), device="cuda", generator=g).to(dtype)
    key, value = fused[:, heads:2 * heads], fused[:, 3 * heads:]
    kc, vc = (make_cache(blocks, heads, block, dim, dtype, layout, fill=7.0) for _ in range(2))
    slots = torch.randperm(blocks * block, device="cuda", generator=g)[:tokens]
    slots[tokens // 2] = -1
    decode.kv_cache_append(key, value, kc, vc, slots)
    for new, cache in ((key, kc), (value, vc)):
        want = torch.full((blocks * block, heads, dim), 7.0, dtype=dtype, device="cuda")
        keep = slots >= 0
        want[slots[keep]] = new[keep]
        assert torch.equal(cache, want.view(blocks, block, heads, dim).permute(0, 2, 1, 3))


@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,block", [(1, 1, 8, 1), (5, 3, 7, 4), (64, 8, 128, 16), (33, 2, 80, 5), (300, 5, 256, 24), (3, 1, 1000, 64)])
def test_append_quantizes_rows_as_the_quantizer_does(decode, tokens, heads, dim, block, dtype, layout):
    from fbgemm_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + dim)
    blocks, row = -(-tokens // block) + 3, decode.kv_row_bytes(dim)
    fused = (torch.randn((tokens, 2 * heads, dim), device="cuda", generator=g) + 0.25).to(dtype)
    fused[0, 0] = 3.0  # a constant row
    key, value = fused[:, :heads], fused[:, heads:]
    kc, vc = (make_cache(blocks, heads, block, row, torch.uint8, layout, fill=9) for _ in range(2))
    slots = torch.randperm(blocks * block, device="cuda", generator=g)[:tokens]
    decode.kv_cache_append(key, value, kc, vc, slots)
    for new, cache in ((key, kc), (value, vc)):
        want = torch.full((blocks * block, heads, row), 9, dtype=torch.uint8, device="cuda")
        rows = ops.quantize_rowwise(new.float().reshape(-1, dim), 8, layout=ops.QLAYOUT_TBE)
        want[slots, :, : dim + 4] = rows.view(tokens, heads, dim + 4)
        assert torch.equal(cache, want.view(blocks, block, heads, row).permute(0, 2, 1, 3))


def test_append_of_numbers_that_the_format_does_not_hold(decode):
    """Elements beyond fp16's largest number count as that one, NaN as 0."""
    x = torch.randn((6, 1, 64), device="cuda")
    x[0, 0, 5], x[1, 0, 6], x[2, 0, 7], x[3, 0, 8], x[4] = float("inf"), -float("inf"), float("nan"), 1e30, float("nan")
    kc, vc = (make_cache(1, 1, 8, 68, torch.uint8, "hnd", fill=0) for _ in range(2))
    from fbgemm_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        new = x.to(dtype)
        decode.kv_cache_append(new, new, kc, vc, torch.arange(6, device="cuda"))
        want = ops.quantize_rowwise(new.float().nan_to_num(nan=0.0).clamp(-65504, 65504).reshape(6, 64), 8, layout=ops.QLAYOUT_TBE)
        assert torch.equal(kc[0, 0, :6], want) and torch.equal(vc, kc)


@pytest.mark.parametrize("dtype,row", [(torch.bfloat16, 64), (torch.uint8, 68)])
def test_append_reports_slots_outside_the_cache(decode, dtype, row):
    from fbgemm_amd import ops
    new = torch.randn((9, 2, 64), device="cuda").bfloat16()
    kc, vc = (make_cache(2, 2, 4, row, dtype, "hnd", fill=1) for _ in range(2))
    st = ops.Status()
    for slots, want in (([0, 1, 2, -1, 3, 4, 5, -1, 6], (0, -1)), ([0, 1, 8, 2, -2, 3, 4, 5, 1 << 40], (1, 2))):
        st.clear()
        decode.kv_cache_append(new, new, kc, vc, torch.tensor(slots, device="cuda"), status=st)
        assert st.read() == want
    assert (kc[1, :, 3] == 1).all()  # the slot that nobody had


# ---- attention --------------------------------------------------------------------------------------


def attention_case(decode, seed, dim, heads, kv_heads, block, lengths, dtype, rows8=False, layout="hnd", poison=True, width=None, index=torch.int32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B = len(lengths)
    used = [-(-max(n, 0) // block) for n in lengths]
    width = width or max(max(used), 1)
    blocks = sum(used) + 2
    pages = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((B, width), 1 << 30, dtype=torch.int32, device="cuda")
    at = 0
    written = torch.zeros((blocks, block), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        tables[b, :used[b]] = pages[at:at + used[b]][:width]
        for j in range(used[b]):
            written[pages[at + j].long(), : min(block, n - j * block)] = True
        at += used[b]
    query = torch.randn((B, heads, dim), device="cuda", generator=g).to(dtype)
    caches, values = [], []
    for _ in range(2):
        if rows8:
            c = make_cache(blocks, kv_heads, block, decode.kv_row_bytes(dim), torch.uint8, layout)
            c.copy_(torch.randint(0, 256, c.shape, device="cuda", generator=g, dtype=torch.uint8))
            scale = 4.0 / 255 * (0.5 + torch.rand((*c.shape[:3], 1), device="cuda", generator=g))
            c[..., :4] = torch.cat((scale, scale * -130 * torch.rand(scale.shape, device="cuda", generator=g)), -1).half().view(torch.uint8)
            if poison:  # scales and biases of rows without a token: NaN
                c.masked_fill_(~written[:, None, :, None], 255)
            values.append(R.rows8_values(c.cpu().numpy(), dim))
        else:
            c = make_cache(blocks, kv_heads, block, dim, dtype, layout)
            c.copy_(torch.randn(c.shape, device="cuda", generator=g))
            if poison:
                c.masked_fill_(~written[:, None, :, None], float("nan"))
                c[:, :, -1:].masked_fill_(~written[:, None, -1:, None], float("inf"))
            values.append(np64(c))
        caches.append(c)
    return query, caches, values, tables, torch.tensor(lengths, device="cuda", dtype=index)


def check_attention(decode, case, dtype, scale=None, window=0, softcap=0.0):
    query, caches, values, tables, lengths = case
    got, lse = decode.paged_attention(query, *caches, tables, lengths, scale=scale, window=window, softcap=softcap)
    assert got.dtype == dtype and got.shape == query.shape and lse.dtype == torch.float32
    s = query.shape[2] ** -0.5 if scale is None else scale
    want, want_lse, off, lse_off = R.attention(np64(query), *values, tables.cpu().numpy(), lengths.cpu().numpy(), s, window, softcap)
    close(got, want, off, dtype)
    close(lse, want_lse, lse_off, torch.float32)
    again = decode.paged_attention(query, *caches, tables, lengths, scale=scale, window=window, softcap=softcap)
    assert torch.equal(again[0], got) and torch.equal(again[1], lse)  # the same bits every time


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257]


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", [1, 7, 16, 24, 48, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_at_the_edges_of_tiles_and_pages(decode, dim, block, dtype, rows8):
    check_attention(decode, attention_case(decode, dim + block, dim, 4, 2, block, EDGES, dtype, rows8), dtype)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 80, 96, 120, 136, 192, 248])
def test_attention_of_dims_between(decode, dim, rows8):
    check_attention(decode, attention_case(decode, dim, dim, 6, 2, 16, [0, 1, 40, 133, 300], torch.bfloat16, rows8), torch.bfloat16)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (6, 2), (7, 1), (15, 1), (16, 1), (17, 1), (32, 2), (66, 2), (40, 1)])
def test_attention_of_shared_heads(decode, heads, kv_heads, rows8):
    check_attention(decode, attention_case(decode, heads, 64, heads, kv_heads, 16, [3, 0, 200, 65], torch.float16, rows8), torch.float16)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("layout", ["nhd", "padded"])
@pytest.mark.parametrize("block", [16, 20])
def test_attention_over_strided_caches(decode, layout, block, rows8):
    case = attention_case(decode, block, 128, 8, 4, block, [150, 33, 1], torch.bfloat16, rows8, layout, index=torch.int64)
    fused = torch.zeros((3, 24, 128), dtype=torch.bfloat16, device="cuda")
    fused[:, 3:11] = case[0]
    check_attention(decode, (fused[:, 3:11], *case[1:]), torch.bfloat16)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("block", [16, 10])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0.0, None), (17, 0.0, 0.3), (128, 5.0, None), (1000, 30.0, 0.5), (0, 2.0, -0.2), (130, 0.0, 0.0)])
def test_attention_with_a_window_a_cap_and_a_scale(decode, window, softcap, scale, block, rows8):
    case = attention_case(decode, window, 128, 4, 2, block, [0, 1, 16, 129, 130, 131, 500], torch.float16, rows8)
    check_attention(decode, case, torch.float16, scale, window, softcap)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("block", [16, 12])
def test_attention_split_over_workers(decode, block, rows8):
    """Long contexts beside short ones: pairs of requests and heads that several workers share, and empty ones between them."""
    case = attention_case(decode, 5, 64, 8, 2, block, [9000, 0, 1, 20011, 0, 128, 4097], torch.bfloat16, rows8)
    check_attention(decode, case, torch.bfloat16)
    check_attention(decode, attention_case(decode, 6, 64, 2, 1, block, [70003], torch.float16, rows8), torch.float16)


def test_attention_of_more_requests_than_a_workgroup_adds_up_at_once(decode):
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 40, 1500).tolist()
    check_attention(decode, attention_case(decode, 7, 64, 3, 3, 16, lengths, torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("block", [16, 10])
def test_attention_leaves_out_blocks_that_are_not_there(decode, block, rows8):
    query, caches, values, tables, lengths = attention_case(decode, 8, 64, 4, 2, block, [100, 64, 31, 16], torch.float16, rows8)
    tables[0, 1], tables[0, 3], tables[1], tables[2, 0] = -1, 1 << 29, -1, caches[0].shape[0]
    check_attention(decode, (query, caches, values, tables, lengths), torch.float16)


def test_attention_of_lengths_beyond_the_table_and_below_zero(decode):
    query, caches, values, tables, lengths = attention_case(decode, 9, 64, 4, 2, 16, [64, 64, 64], torch.float16)
    check_attention(decode, (query, caches, values, tables, torch.tensor([-4, 1000, 1 << 40], device="cuda")), torch.float16)
    empty = [c[:0] for c in caches]
    out, lse = decode.paged_attention(query, *empty, tables, lengths)
    assert (out == 0).all() and (lse == -float("inf")).all()
    out, lse = decode.paged_attention(query, *caches, tables[:, :0], lengths)
    assert (out == 0).all() and (lse == -float("inf")).all()
    out, lse = decode.paged_attention(query[:0], *caches, tables[:0], lengths[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_attention_of_scores_far_apart(decode):
    """Maxima that move late and by much, and scores so far below the maximum that their weights are zero."""
    query, caches, values, tables, lengths = attention_case(decode, 10, 64, 4, 2, 16, [700, 300], torch.bfloat16, poison=False)
    for c in caches[:1]:
        c[:, :, ::5] *= 40
    values[0] = np64(caches[0])
    check_attention(decode, (query, caches, values, tables, lengths), torch.bfloat16)


def test_attention_beyond_32_bit_offsets(decode):
    """Pages of a cache of 5 GiB, the last ones among them."""
    blocks, block = 20480, 64
    kc, vc = (torch.zeros((blocks, 8, block, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pages = [blocks - 1, 3, blocks // 2 + 1, 16384]
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    query = torch.randn((1, 16, 128), device="cuda", generator=g).bfloat16()
    rows = torch.randn((2, 200, 8, 128), device="cuda", generator=g).bfloat16()
    slots = torch.tensor([pages[t // block] * block + t % block for t in range(200)], device="cuda")
    decode.kv_cache_append(rows[0], rows[1], kc, vc, slots)
    got, lse = decode.paged_attention(query, kc, vc, torch.tensor([pages], dtype=torch.int32, device="cuda"), torch.tensor([200], device="cuda"))
    small = [np64(r).reshape(1, 200, 8, 128).transpose(0, 2, 1, 3) for r in rows]
    want, want_lse, off, lse_off = R.attention(np64(query), *small, np.zeros((1, 1), np.int64), np.array([200]), 128 ** -0.5)
    close(got, want, off, torch.bfloat16)
    close(lse, want_lse, lse_off, torch.float32)


# ---- logits -----------------------------------------------------------------------------------------


def logits_case(seed, rows, vocab, history, biases, mask, dtype, index):
    rng = np.random.default_rng(seed)
    count = rng.integers(0, history + 1, rows)
    count[0] = history
    if rows > 1:
        count[1] = 0
    offsets = np.concatenate([[0], np.cumsum(count)])
    tokens = (vocab * rng.uniform(0, 1, offsets[-1]) ** 3).astype(index)
    tokens[::17] = vocab + 5  # not of the vocabulary: passed over
    tokens[::19] = -1
    prompts = (count * rng.uniform(0, 1, rows)).astype(index)
    x = torch.from_numpy(4 * rng.standard_normal((rows, vocab)).astype(np.float32)).to(dtype)
    f32 = lambda a: a.astype(np.float32)
    each = biases * rows
    ids = rng.integers(-1, vocab + 1, each).astype(index)
    if each > 3:
        ids[1] = ids[3] = ids[0] = vocab - 1  # several for one token: the last one counts
    return dict(x=x, tokens=tokens, offsets=offsets.astype(index), prompts=prompts, repetition=f32(rng.uniform(0.8, 1.5, rows)),
                frequency=f32(rng.uniform(-0.5, 1, rows)), presence=f32(rng.uniform(0, 1, rows)),
                bias_ids=ids if biases else None, bias_values=f32(rng.uniform(-2, 2, each)) if biases else None,
                bias_offsets=(np.arange(rows + 1) * biases).astype(index) if biases else None,
                mask=rng.integers(-(1 << 31), 1 << 31, (rows, (vocab + 31) // 32)).astype(np.int32) if mask else None)


def check_logits(decode, c, logits=None, out=None):
    dtype = c["x"].dtype
    dev = {k: None if v is None else (v.cuda() if torch.is_tensor(v) else cu(v)) for k, v in c.items()}
    logits = dev.pop("x") if logits is None else logits
    dev.pop("x", None)
    want, off = R.logits(np64(c["x"]), *[c[k] for k in ("tokens", "offsets", "prompts", "repetition", "frequency", "presence", "bias_ids", "bias_values", "bias_offsets", "mask")])
    got = decode.penalize_logits(logits, dev["tokens"], dev["offsets"], dev["prompts"], repetition=dev["repetition"], frequency=dev["frequency"],
                                 presence=dev["presence"], bias_ids=dev["bias_ids"], bias_values=dev["bias_values"],
                                 bias_offsets=dev["bias_offsets"], mask=dev["mask"], out=out)
    assert got.dtype == dtype
    close(got, want, off, dtype)
    return got


@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 3, 1, True), (2, 31, 40, 0, True), (3, 33, 0, 4, False), (4, 8191, 500, 5, True), (5, 8193, 3000, 0, False), (2, 40_001, 70_000, 300, True),
    (2, 6000, 900, 2047, True), (3, 6000, 900, 2048, False), (1, 5000, 1_060_000, 7, True)])
def test_logits(decode, rows, vocab, history, biases, mask, dtype, index):
    check_logits(decode, logits_case(vocab, rows, vocab, history, biases, mask, dtype, index))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_in_place_and_of_strided_rows(decode, dtype):
    c = logits_case(5, 3, 9001, 100, 3, True, dtype, np.int64)
    wide = torch.full((3, 9050), 5.0, dtype=dtype, device="cuda")
    view = wide[:, 13:9014]
    view.copy_(c["x"])
    got = check_logits(decode, c, logits=view, out=view)
    assert got.data_ptr() == view.data_ptr() and (wide[:, :13] == 5).all() and (wide[:, 9014:] == 5).all()


def test_logits_with_parts_left_out(decode):
    full = logits_case(6, 3, 5000, 200, 4, True, torch.float16, np.int32)
    for leave in (("prompts",), ("repetition",), ("frequency", "presence"), ("mask",), ("bias_ids", "bias_values", "bias_offsets"),
                  ("tokens", "offsets", "prompts"), ("tokens", "offsets", "prompts", "bias_ids", "bias_values", "bias_offsets"),
                  ("tokens", "offsets", "prompts", "bias_ids", "bias_values", "bias_offsets", "mask")):
        check_logits(decode, {k: None if k in leave else v for k, v in full.items()})


def test_logits_that_are_not_finite_and_rows_that_a_mask_empties(decode):
    c = logits_case(7, 2, 100, 30, 2, True, torch.float32, np.int64)
    c["x"][0, ::3], c["x"][0, 1::3] = float("nan"), float("inf")
    c["mask"][:] = 0
    got = check_logits(decode, c)  # whatever is behind the mask
    assert (got == -float("inf")).all()
    c["mask"][:] = -1
    c["x"][0, ::3], c["x"][0, 1::3] = torch.finfo(torch.float32).min, -float("inf")
    c["bias_values"][:] = 0
    c["frequency"][:] = c["presence"][:] = 0
    c["repetition"][:] = 1
    assert torch.equal(check_logits(decode, c).cpu(), c["x"])


# ---- together ---------------------------------------------------------------------------------------


def step(decode, s):
    t = decode.kv_block_tables(s["lengths"], s["new"], s["tables"], s["free"], s["start"], 16, len(s["key"]))
    decode.kv_cache_append(s["key"], s["value"], s["kc"], s["vc"], t.slots)
    out, lse = decode.paged_attention(s["query"], s["kc"], s["vc"], s["tables"], t.lengths)
    logits = decode.penalize_logits(s["logits"], s["tokens"], s["offsets"], frequency=s["frequency"])
    return (*t, out, lse, logits, s["tables"].clone(), s["kc"].clone())


def step_state(seed, rows8):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B = 5
    lengths = torch.tensor([0, 16, 31, 300, 77], device="cuda", dtype=torch.int32)
    pages = torch.randperm(60, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((B, 24), -1, dtype=torch.int32, device="cuda")
    used = (lengths + 15) // 16
    tables[torch.arange(24, device="cuda") < used[:, None]] = pages[: int(used.sum())]
    rows = lambda *shape: torch.randn(shape, device="cuda", generator=g)
    s = dict(lengths=lengths, new=torch.ones_like(lengths), tables=tables, free=pages, start=used.sum().to(torch.int32).reshape(1),
             key=rows(B, 2, 64).bfloat16(), value=rows(B, 2, 64).bfloat16(), query=rows(B, 8, 64).bfloat16(), logits=rows(B, 4000),
             tokens=torch.randint(0, 4000, (100,), device="cuda", generator=g), offsets=torch.arange(B + 1, device="cuda") * 20,
             frequency=torch.full((B,), 0.5, device="cuda"))
    for name in ("kc", "vc"):
        if rows8:
            s[name] = torch.randint(0, 60, (60, 2, 16, 68), device="cuda", generator=g, dtype=torch.uint8)
        else:
            s[name] = rows(60, 2, 16, 64).bfloat16()
    return s


@pytest.mark.parametrize("rows8", [False, True])
def test_a_captured_step_replays_and_follows_its_inputs(decode, rows8):
    s, want = step_state(1, rows8), []
    others = [step_state(k, rows8) for k in (2, 3, 4)]
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


def test_a_step_on_another_stream(decode):
    s = step_state(5, False)
    want = step(decode, {k: v.clone() for k, v in s.items()})
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(decode, s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(decode):
    s = step_state(6, False)
    s8 = step_state(6, True)
    cpu = {k: v.cpu() for k, v in s.items()}
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)  # rows off their boundary
    tables = lambda **k: decode.kv_block_tables(*[{**s, **k}[n] for n in ("lengths", "new", "tables", "free", "start")], k.get("block", 16), k.get("n", 5))
    append = lambda **k: decode.kv_cache_append(*[{**s, "slots": torch.arange(5, device="cuda"), **k}[n] for n in ("key", "value", "kc", "vc", "slots")])
    attend = lambda kw={}, **k: decode.paged_attention(*[{**s, **k}[n] for n in ("query", "kc", "vc", "tables", "lengths")], **kw)
    penalize = lambda **k: decode.penalize_logits({**s, **k}["logits"], **{n: v for n, v in k.items() if n != "logits"})
    refused = [
        lambda: tables(lengths=s["lengths"].float()), lambda: tables(new=s["new"].long()), lambda: tables(new=s["new"][:4]),
        lambda: tables(tables=s["tables"].long()), lambda: tables(tables=s["tables"][:4]), lambda: tables(tables=s["tables"].t()),
        lambda: tables(free=s["free"].long()), lambda: tables(start=s["free"]), lambda: tables(start=cpu["start"]), lambda: tables(block=0),
        lambda: tables(n=-1), lambda: tables(lengths=s["free"][::12], new=s["new"]),
        lambda: append(key=s["key"].half()), lambda: append(key=s["key"][:4]), lambda: append(value=s["value"].half(), key=s["key"].half()),
        lambda: append(key=s["key"].transpose(1, 2), value=s["value"].transpose(1, 2)), lambda: append(slots=torch.arange(4, device="cuda")),
        lambda: append(slots=torch.arange(5, device="cuda", dtype=torch.int32)), lambda: append(kc=s["kc"][:, :1], vc=s["vc"][:, :1]),
        lambda: append(kc=s["kc"], vc=s["vc"][:3]), lambda: append(kc=s["kc"][0], vc=s["vc"][0]), lambda: append(slots=torch.arange(5)),
        lambda: append(kc=s8["kc"][..., :60], vc=s8["vc"][..., :60]), lambda: append(kc=odd(s8["kc"]), vc=s8["vc"]),
        lambda: append(key=s["key"].double(), value=s["value"].double(), kc=s["kc"].double(), vc=s["vc"].double()),
        lambda: append(kc=torch.zeros((4, 2, 16, 69), dtype=torch.uint8, device="cuda"), vc=torch.zeros((4, 2, 16, 69), dtype=torch.uint8, device="cuda")),
        lambda: attend(query=s["query"].half()), lambda: attend(query=s["query"].float()), lambda: attend(query=s["query"][:, :7]),
        lambda: attend(query=s["query"][..., :60], kc=s["kc"][..., :60], vc=s["vc"][..., :60]), lambda: attend(query=s["query"][0]),
        lambda: attend(query=odd(s["query"])), lambda: attend(kc=odd(s["kc"])), lambda: attend(tables=s["tables"].long()),
        lambda: attend(tables=s["tables"][:4]), lambda: attend(lengths=s["lengths"].float()), lambda: attend(lengths=s["lengths"][:4]),
        lambda: attend(lengths=cpu["lengths"]), lambda: attend(kw={"window": -1}), lambda: attend(kw={"softcap": -1.0}),
        lambda: attend(kw={"scale": float("nan")}), lambda: attend(kw={"softcap": float("inf")}), lambda: attend(kc=s["kc"].half(), vc=s["vc"].half()),
        lambda: attend(query=torch.zeros((5, 8, 264), dtype=torch.bfloat16, device="cuda"), kc=torch.zeros((4, 2, 16, 264), dtype=torch.bfloat16, device="cuda"),
                       vc=torch.zeros((4, 2, 16, 264), dtype=torch.bfloat16, device="cuda")),
        lambda: penalize(logits=s["logits"].double()), lambda: penalize(logits=s["logits"][0]), lambda: penalize(logits=s["logits"].t()),
        lambda: penalize(tokens=s["tokens"]), lambda: penalize(tokens=s["tokens"], offsets=s["offsets"].int()), lambda: penalize(offsets=s["offsets"]),
        lambda: penalize(tokens=s["tokens"], offsets=s["offsets"][:4]), lambda: penalize(prompt_lengths=s["lengths"].long()),
        lambda: penalize(repetition=s["frequency"][:4]), lambda: penalize(repetition=s["frequency"].double()), lambda: penalize(repetition=cpu["frequency"]),
        lambda: penalize(bias_ids=s["tokens"]), lambda: penalize(bias_ids=s["tokens"], bias_values=s["logits"][0, :99], bias_offsets=s["offsets"]),
        lambda: penalize(mask=torch.zeros((5, 124), dtype=torch.int32, device="cuda")), lambda: penalize(mask=torch.zeros((5, 125), dtype=torch.int64, device="cuda")),
        lambda: penalize(out=s["logits"].half()), lambda: penalize(out=s["logits"][:, :100]),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError, TypeError, NotImplementedError)):
            call()
            print("not refused:", i)
    # none of them left an error behind for what runs next
    step(decode, s)
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError):  # no CPU path
        decode.paged_attention(*[cpu[n] for n in ("query", "kc", "vc", "tables", "lengths")])


@pytest.mark.parametrize("rows8", [False, True])
def test_attention_on_two_streams_at_once(decode, rows8):
    """Calls whose pairs are shared by many workers, side by side: each stream joins its own."""
    cases = [attention_case(decode, 20 + k, 64, 2, 1, 16, [30011, 5, 4099], torch.bfloat16, rows8) for k in range(2)]
    want = [decode.paged_attention(q, *c, t, n) for q, c, _, t, n in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                q, c, _, t, n = cases[k]
                got[k].append(decode.paged_attention(q, *c, t, n))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for pair in got[k] for a, b in zip(pair, want[k]))


def test_attention_call_behind_call(decode):
    """Calls of other inputs one behind the other, nothing waiting between: each one's sums are its own, though their scratch is one."""
    cases = [attention_case(decode, 40 + k, 64, 4, 2, 16, lengths, torch.bfloat16, rows8)
             for k, (lengths, rows8) in enumerate((([20011, 300, 5], False), ([77, 9000, 4099], False), ([12345], True), ([1, 30003], True)))]
    call = lambda case: decode.paged_attention(case[0], *case[1], case[3], case[4])  # noqa: E731
    want = []
    for case in cases:
        want.append(call(case))
        torch.cuda.synchronize()
    for order in ((0, 1, 0, 1, 2, 3, 2, 0), (3, 2, 1, 0, 0, 3, 1, 2)):
        got = [(k, call(cases[k])) for k in order for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for k, pair in got for a, b in zip(pair, want[k]))


def test_attention_in_many_captures(decode):
    """Many captures, replayed out of order, beside eager calls."""
    q, c, _, t, n = attention_case(decode, 30, 64, 2, 1, 16, [9001, 70], torch.bfloat16)
    want = decode.paged_attention(q, *c, t, n)
    graphs = []
    for _ in range(20):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [decode.paged_attention(q, *c, t, n) for _ in range(2)]
        graphs.append((graph, got))
    for k in (3, 19, 0, 7, 3, 0):
        eager = decode.paged_attention(q, *c, t, n)
        graphs[k][0].replay()
        torch.cuda.synchronize()
        for pair in [eager, *graphs[k][1]]:
            assert all(torch.equal(a, b) for a, b in zip(pair, want))


@pytest.mark.parametrize("rows8", [False, True])
def test_the_example_generates_what_a_dense_layer_does(rows8):
    """Logits of the paged path against the dense layer: attention's outputs round to bf16 in both (2^-8 of each number, two
    products behind them average it out), 8-bit rows are off by half a step of 1/255 of a row's range, some 6 standard deviations."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    said, lengths, logits, d = example.generate(requests=5, steps=20, rows8=rows8)
    for r in range(5):
        n = int(lengths[r])
        assert (said[r, :n] >= 0).all() and (said[r, n:] == -1).all()
        want = example.dense_logits(d, said[r, :n - 1]).float()
        off = float((logits[r].float() - want).norm() / want.norm())
        assert off < (0.05 if rows8 else 0.02), off
