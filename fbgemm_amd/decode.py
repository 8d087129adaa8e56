"""A decoding step over a paged key-value cache: block tables, rotary positions, cache rows, attention, logits, sampling.

What a server of a language model runs for every new token of many requests at once, next to the embedding lookups of
``ops``. The operators have no counterpart in the reference's quantized-embedding path; they keep its manner: lists are
(indices, offsets) pairs on the device, 8-bit and 4-bit cache rows are the table-batched operator's (fp16 scale and bias in front),
input errors are recorded in an ``ops.Status`` block where one is given.

A cache is two tensors ``[blocks, heads, block_size, row]``, keys and values, with any strides of the first three
dimensions: fp16 or bf16 rows of ``dim`` elements, or uint8 rows of ``kv_row_bytes(dim, row_bits)`` bytes, whose elements have
8 bits, or 4 where ``row_bits=4`` says so.

One step::

    t = kv_block_tables(lengths, new_tokens, block_tables, free_blocks, free_start, block_size, num_tokens)
    query, key = rotate_positions(query, key, t.positions, frequencies)
    kv_cache_append(key, value, key_cache, value_cache, t.slots)
    out, lse = paged_attention(query, key_cache, value_cache, block_tables, t.lengths)
    logits = penalize_logits(logits, tokens, offsets, prompt_lengths, repetition=..., mask=...)
    tokens, log_probabilities = sample_tokens(logits, torch.rand(...), temperature=..., top_p=...)

and ``t.lengths`` and ``t.free_start`` are the next step's. Everything stays on the device and on the current stream:
nothing waits, and a step can be captured into a graph. ``examples/paged_decode.py`` runs one.

All tensors are device tensors; everything runs in the HIP library (the operators ``torch.ops.fbgemm_amd.*``, which these
functions call), nothing here computes. It is for inference: of them ``rotate_positions`` alone has a gradient.
"""
import collections
import math
import os

import torch

from .build import TORCH_OP_OUT
from .ops import Status  # noqa: F401  (the block that `status` arguments take)

if not os.path.exists(TORCH_OP_OUT):
    raise RuntimeError(f"{TORCH_OP_OUT} is missing: build it with `python -m fbgemm_amd.build`. There is no CPU fallback.")
torch.ops.load_library(TORCH_OP_OUT)

BlockTables = collections.namedtuple("BlockTables", "slots positions offsets lengths free_start")
Samples = collections.namedtuple("Samples", "tokens log_probabilities")

ERR_OUT_OF_BLOCKS = 16  # kv_block_tables: the free list has no block left for a token

_op = torch.ops.fbgemm_amd
_block_tables = _op.kv_block_tables.default
_append = _op.kv_cache_append.default
_attention = _op.paged_attention.default
_penalize = _op.penalize_logits.default
_penalize_out = _op.penalize_logits.out
_read = _op.kv_cache_read.default
_rotate = _op.rotate_positions.default
_rotate_out = _op.rotate_positions.out
_sample = _op.sample_tokens.default


def kv_row_bytes(dim, row_bits=8):
    """Bytes of an 8-bit or 4-bit cache row: fp16 scale, fp16 bias, ``dim`` codes, on a 4-byte boundary."""
    if row_bits not in (8, 4):
        raise ValueError(f"row_bits must be 8 or 4, got {row_bits}")
    if row_bits == 4 and dim % 2:
        raise ValueError(f"4-bit rows hold an even number of elements, got {dim}")
    return (dim * row_bits // 8 + 4 + 3) // 4 * 4


def rotary_frequencies(dim, base=10_000.0, factor=1.0, trained=None, low=1.0, high=4.0, device="cuda"):
    """Frequencies of ``rotate_positions`` for ``dim`` turned elements: ``base ** (-2 p / dim)`` radians a position, fp64 ``[dim / 2]``.

    For contexts ``factor`` times longer than a model's: all divided by it, or, with ``trained`` (the positions the model knows),
    only those of waves longer than ``trained / low``; those of waves shorter than ``trained / high`` are kept, and between
    the two the kept part grows with the number of waves in ``trained``. A model's weights go with its frequencies: they are
    made once."""
    if dim <= 0 or dim % 2:
        raise ValueError(f"an even number of elements is turned, got {dim}")
    if not (base > 0 and factor > 0) or (trained is not None and not (trained > 0 and high > low)):
        raise ValueError("base, factor and trained must be positive, high larger than low")
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if trained is None:
        f = f / factor
    else:
        kept = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (kept + (1 - kept) / factor)
    return f.to(device)


def kv_block_tables(lengths, new_tokens, block_tables, free_blocks, free_start, block_size, num_tokens, status=None):
    """Blocks for the tokens a step adds, and their slots, from the requests' lengths.

    ``lengths`` and ``new_tokens`` (int32 or int64, ``[requests]``): tokens a request holds, and gets. ``block_tables``
    (int32 ``[requests, width]``, written in place): the entries behind a request's own get the next blocks of
    ``free_blocks`` (int32) from ``free_start`` (int32, one entry) on, requests in order. ``num_tokens``: the sum of
    ``new_tokens``, or more where the step's tensors are padded.

    Returns ``BlockTables``: ``slots`` (int64 ``[num_tokens]``, -1 where there is no block) and ``positions`` (int64) of the
    new tokens, request by request, ``offsets`` (int32 ``[requests + 1]``) of the requests in them, ``lengths`` with the new
    tokens, and the next ``free_start`` (beyond ``len(free_blocks)`` by as many blocks as are missing). The inputs but
    ``block_tables`` are left as they are, so the same call gives the same again.

    ``status`` records ``ERR_NEGATIVE_LENGTH`` (counted as 0), ``ERR_BAG_OVERRUN`` (a table too narrow for its tokens),
    ``ERR_OUT_OF_BLOCKS`` and ``ERR_LENGTH_MISMATCH`` (``num_tokens`` is not the sum). A step that is padded on purpose records the
    last too: it is told from a list that was cut by ``offsets[-1]``, which is below ``num_tokens`` then. Positions of a request that
    holds more than its table has room for count from the table's room; their slots are -1."""
    return BlockTables._make(_block_tables(lengths, new_tokens, block_tables, free_blocks, free_start, block_size, num_tokens,
                                           None if status is None else status.buf))


def rotate_positions(query, key, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False, out=None):
    """Queries and keys (``[tokens, heads, dim]`` each, fp32, fp16 or bf16) turned by their tokens' ``positions`` (int32 or int64).

    Of the first ``2 * len(frequencies)`` elements of a head, pair ``p`` is ``(p, p + len(frequencies))``, or with ``interleaved``
    ``(2 p, 2 p + 1)``: ``(a, b)`` becomes ``magnitude * (a cos - b sin, b cos + a sin)`` of ``positions * frequencies[p]`` (fp64,
    ``rotary_frequencies``); the elements behind them stay as they are. Angles are taken in fp64, products in fp32, rounded once.
    With ``inverse`` the other way round, with the same magnitude: what a gradient goes through, or a key that gives up its position.

    Returns new tensors, through which gradients go to ``query`` and ``key``, or ``out``, a pair, which may be ``(query, key)``; nothing
    else that is read may overlap it. Into ``out`` there is no gradient: a call that would need one is refused (``torch.no_grad()``)."""
    if out is None:
        return _rotate(query, key, positions, frequencies, interleaved, magnitude, inverse)
    return _rotate_out(query, key, positions, frequencies, interleaved, magnitude, inverse, query_out=out[0], key_out=out[1])


def kv_cache_append(key, value, key_cache, value_cache, slots, status=None, row_bits=8):
    """Write the rows of new tokens, ``key`` and ``value`` ``[tokens, heads, dim]``, to their ``slots`` (int64) of the cache.

    fp32, fp16 and bf16 caches take rows of their own type as they are; a uint8 cache takes any of the three and holds
    what ``ops.quantize_rowwise(rows, row_bits, layout=QLAYOUT_TBE)`` makes of them (elements beyond fp16's range at its end, NaN as
    0; of 4 bits an even number).
    A token of slot -1 is skipped, and one whose slot the cache does not have: that one is recorded in ``status``
    (``ERR_INDEX_OUT_OF_RANGE`` and its number). Slots differ from each other, but for -1: what a slot holds that several tokens have
    is a mixture of theirs. Key and value may be slices of a fused projection's output; the caches' rows must not overlap."""
    _append(key, value, key_cache, value_cache, slots, None if status is None else status.buf, row_bits)


def kv_cache_read(key_cache, value_cache, block_tables, offsets, num_tokens, dim, dtype=None, starts=None, status=None, row_bits=8):
    """The rows of requests' tokens out of their pages: keys and values ``[num_tokens, heads, dim]``, for attention of a prompt's later
    part over its earlier one, or to move requests.

    Token ``i`` is that of request ``r`` with ``offsets[r] <= i < offsets[r + 1]`` (int32 or int64 ``[requests + 1]``, ascending) at
    position ``starts[r] + i - offsets[r]`` (``starts``: like ``offsets``, by default 0). fp32, fp16 and bf16 rows come as they are; 8-bit
    and 4-bit ones as the values they stand for, ``scale * code + bias`` in fp32, rounded once to ``dtype`` (by default fp32).

    Tokens whose block the table or the cache does not have are zeros and recorded in ``status`` (``ERR_INDEX_OUT_OF_RANGE`` and the
    first one's number); tokens from ``offsets[-1]`` on are zeros."""
    return _read(key_cache, value_cache, block_tables, offsets, num_tokens, dim, dtype, starts, None if status is None else status.buf, row_bits)


def paged_attention(query, key_cache, value_cache, block_tables, lengths, scale=None, window=0, softcap=0.0, row_bits=8):
    """Attention of one new token per request over its tokens in the cache.

    ``query`` fp16 or bf16 ``[requests, query_heads, dim]`` (``query_heads`` a multiple of the cache's heads: that many
    queries in a row share one; ``dim`` a multiple of 8, at most 256), the cache 16-bit rows of the same type or uint8
    rows of ``row_bits``; ``lengths`` (int32 or int64) counts the new token too. ``scale`` of the scores, by default ``dim ** -0.5``;
    ``window`` > 0: the last that many tokens only; ``softcap`` > 0: scores ``s`` become ``softcap * tanh(s / softcap)``.

    Returns the outputs (the queries' type and shape) and the logarithm of each softmax's sum (fp32 ``[requests,
    query_heads]``), by which results over several caches can be joined. Tokens of a block that the cache does not have
    are left out; where none is left the output is 0 and the logarithm -inf. Rows without a token are never looked at for their
    contents; a token's NaN reaches its queries' outputs, a score of -inf weighs nothing."""
    return _attention(query, key_cache, value_cache, block_tables, lengths, scale, window, softcap, row_bits)


def penalize_logits(logits, tokens=None, offsets=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
                    bias_ids=None, bias_values=None, bias_offsets=None, mask=None, out=None):
    """Penalties for the tokens of a row, biases and a grammar's mask on ``logits`` ``[rows, vocab]`` (fp32, fp16, bf16).

    ``tokens`` and ``offsets``: each row's tokens so far, one list of int32 or int64, the first ``prompt_lengths`` of a row
    its prompt's. ``repetition``, ``frequency``, ``presence``: fp32 ``[rows]``, or None for none. A token of the list is
    divided by ``repetition`` (multiplied where it is not positive), one that was said behind the prompt loses ``frequency``
    for every time and ``presence`` once. ``bias_ids``, ``bias_values``, ``bias_offsets``: added to single tokens (of several
    for one the last counts). ``mask``: int32 ``[rows, ceil(vocab / 32)]``, a token whose bit is 0 becomes -inf;
    one row of it may be expanded over all.

    In fp32, rounded once. Returns a new tensor, or ``out``, which may be ``logits``."""
    if out is None:
        return _penalize(logits, tokens, offsets, prompt_lengths, repetition, frequency, presence, bias_ids, bias_values, bias_offsets, mask)
    return _penalize_out(logits, tokens, offsets, prompt_lengths, repetition, frequency, presence, bias_ids, bias_values, bias_offsets, mask, out=out)


def sample_tokens(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """A token of every row of ``logits`` ``[rows, vocab]`` (fp32, fp16, bf16; ``vocab`` at most 2 ** 20), drawn by ``uniform`` (fp32
    ``[rows]``, numbers in [0, 1)).

    With tokens in order, larger logits first and equal ones by number, and ``w = exp((x - max) / temperature)``, those that may be
    drawn are the first ``top_k`` (int32); of these the fewest first ones whose ``w`` add up to ``top_p`` of the sum of all of these; of these the
    ones with ``w >= min_p``. The token is the first of them, by number, where the running sum of ``w`` is above ``uniform`` of
    the whole. Each of the four is ``[rows]`` (fp32 but for ``top_k``) or None for none; ``top_k <= 0``, ``top_p >= 1`` and ``min_p <= 0``
    are none too, and a ``temperature`` or ``top_p`` that is not above 0 is the first of the largest logits, of probability 1.

    NaN and -inf are never drawn, +inf counts as the largest finite number; a row with nothing else gives -1 and -inf. Sums
    are of whole numbers, the same on every run: ``w`` rounded to units of ``2 ** -min(50, 62 - vocab.bit_length())`` of the largest (2 ** -45
    for 131 071 tokens, 2 ** -41 for 2 ** 20), half a unit a token. No gradient goes through it. Returns ``Samples``: ``tokens``
    (int64) and ``log_probabilities`` (fp32), the logarithm of the probability a token was drawn with."""
    return Samples._make(_sample(logits, uniform, temperature, top_k, top_p, min_p))
