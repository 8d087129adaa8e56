"""A decoding step over a paged key-value cache: block tables, cache rows, attention, logits.

What a server of a language model runs for every new token of many requests at once, next to the embedding lookups of
``ops``. The operators have no counterpart in the reference's quantized-embedding path; they keep its manner: lists are
(indices, offsets) pairs on the device, 8-bit cache rows are the table-batched operator's (fp16 scale and bias in front),
input errors are recorded in an ``ops.Status`` block where one is given.

A cache is two tensors ``[blocks, heads, block_size, row]``, keys and values, with any strides of the first three
dimensions: fp16 or bf16 rows of ``dim`` elements, or uint8 rows of ``kv_row_bytes(dim)`` bytes.

One step::

    t = kv_block_tables(lengths, new_tokens, block_tables, free_blocks, free_start, block_size, num_tokens)
    kv_cache_append(key, value, key_cache, value_cache, t.slots)
    out, lse = paged_attention(query, key_cache, value_cache, block_tables, t.lengths)
    logits = penalize_logits(logits, tokens, offsets, prompt_lengths, repetition=..., mask=...)

and ``t.lengths`` and ``t.free_start`` are the next step's. Everything stays on the device and on the current stream:
nothing waits, and a step can be captured into a graph. ``examples/paged_decode.py`` runs one.

All tensors are device tensors; everything runs in the HIP library (the operators ``torch.ops.fbgemm_amd.*``, which these
functions call), nothing here computes.
"""
import collections
import os

import torch

from .build import TORCH_OP_OUT
from .ops import Status  # noqa: F401  (the block that `status` arguments take)

if not os.path.exists(TORCH_OP_OUT):
    raise RuntimeError(f"{TORCH_OP_OUT} is missing: build it with `python -m fbgemm_amd.build`. There is no CPU fallback.")
torch.ops.load_library(TORCH_OP_OUT)

BlockTables = collections.namedtuple("BlockTables", "slots positions offsets lengths free_start")

ERR_OUT_OF_BLOCKS = 16  # kv_block_tables: the free list has no block left for a token

_op = torch.ops.fbgemm_amd
_block_tables = _op.kv_block_tables.default
_append = _op.kv_cache_append.default
_attention = _op.paged_attention.default
_penalize = _op.penalize_logits.default
_penalize_out = _op.penalize_logits.out


def kv_row_bytes(dim):
    """Bytes of an 8-bit cache row: fp16 scale, fp16 bias, ``dim`` bytes, on a 4-byte boundary."""
    return (dim + 4 + 3) // 4 * 4


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


def kv_cache_append(key, value, key_cache, value_cache, slots, status=None):
    """Write the rows of new tokens, ``key`` and ``value`` ``[tokens, heads, dim]``, to their ``slots`` (int64) of the cache.

    fp32, fp16 and bf16 caches take rows of their own type as they are; a uint8 cache takes any of the three and holds
    what ``ops.quantize_rowwise(rows, 8, layout=QLAYOUT_TBE)`` makes of them (elements beyond fp16's range at its end, NaN as 0).
    A token of slot -1 is skipped, and one whose slot the cache does not have: that one is recorded in ``status``
    (``ERR_INDEX_OUT_OF_RANGE`` and its number). Slots differ from each other, but for -1: what a slot holds that several tokens have
    is a mixture of theirs. Key and value may be slices of a fused projection's output; the caches' rows must not overlap."""
    _append(key, value, key_cache, value_cache, slots, None if status is None else status.buf)


def paged_attention(query, key_cache, value_cache, block_tables, lengths, scale=None, window=0, softcap=0.0):
    """Attention of one new token per request over its tokens in the cache.

    ``query`` fp16 or bf16 ``[requests, query_heads, dim]`` (``query_heads`` a multiple of the cache's heads: that many
    queries in a row share one; ``dim`` a multiple of 8, at most 256), the cache 16-bit rows of the same type or uint8
    rows; ``lengths`` (int32 or int64) counts the new token too. ``scale`` of the scores, by default ``dim ** -0.5``;
    ``window`` > 0: the last that many tokens only; ``softcap`` > 0: scores ``s`` become ``softcap * tanh(s / softcap)``.

    Returns the outputs (the queries' type and shape) and the logarithm of each softmax's sum (fp32 ``[requests,
    query_heads]``), by which results over several caches can be joined. Tokens of a block that the cache does not have
    are left out; where none is left the output is 0 and the logarithm -inf. Rows without a token are never looked at for their
    contents; a token's NaN reaches its queries' outputs, a score of -inf weighs nothing."""
    return _attention(query, key_cache, value_cache, block_tables, lengths, scale, window, softcap)


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
