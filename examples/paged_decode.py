"""A small decoder that generates tokens for several requests at once, on the framework's operators.

Token embeddings are rows of a 4-bit table looked up without pooling (``ops.int_nbit_split_embedding_codegen_lookup_function``);
one attention layer keeps its keys and values in a paged cache (``decode.kv_block_tables``, ``kv_cache_append``,
``paged_attention``); the next token is the most likely one behind ``decode.penalize_logits``. The weights are random: what
comes out means nothing, but every request's tokens are those that a dense computation of the same layer gives.

    python examples/paged_decode.py [--rows8] [--requests 6] [--steps 24]

A step reads nothing back: lengths, tables, the free list's place and the tokens stay on the device.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fbgemm_amd import decode, ops  # noqa: E402

VOCAB, DIM, HEADS, KV_HEADS, HEAD_DIM, BLOCK = 4000, 256, 8, 2, 64, 16


class Decoder:
    def __init__(self, requests, longest, rows8, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
        # the table: 4-bit rows in the table-batched operator's layout
        self.row_bytes = ops.padded_row_size_in_bytes(DIM, ops.INT4, 16)
        rows = torch.zeros((VOCAB, self.row_bytes), dtype=torch.uint8, device="cuda")
        ops.quantize_rowwise(normal(VOCAB, DIM), 4, layout=ops.QLAYOUT_TBE, out=rows)
        self.table = rows.view(-1)
        meta = lambda v, dtype: torch.tensor(v, dtype=dtype, device="cuda")  # noqa: E731
        self.placements, self.weights_offsets = meta([0], torch.int32), meta([0], torch.int64)
        self.weights_tys, self.D_offsets = meta([ops.INT4], torch.uint8), meta([0, DIM], torch.int32)
        self.no_uvm = torch.zeros(0, dtype=torch.uint8, device="cuda")
        self.w_qkv = (normal(DIM, (HEADS + 2 * KV_HEADS) * HEAD_DIM) / DIM ** 0.5).bfloat16()
        self.w_out = (normal(HEADS * HEAD_DIM, DIM) / DIM ** 0.5).bfloat16()
        self.w_vocab = (normal(DIM, VOCAB) / DIM ** 0.5).bfloat16()
        # the cache and its pages
        blocks = requests * (-(-longest // BLOCK) + 1)
        if rows8:
            shape, dtype = (blocks, KV_HEADS, BLOCK, decode.kv_row_bytes(HEAD_DIM)), torch.uint8
        else:
            shape, dtype = (blocks, KV_HEADS, BLOCK, HEAD_DIM), torch.bfloat16
        self.key_cache, self.value_cache = torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda")
        self.block_tables = torch.full((requests, -(-longest // BLOCK)), -1, dtype=torch.int32, device="cuda")
        self.free_blocks = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
        self.free_start = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def embed(self, tokens):
        offsets = torch.tensor([0, tokens.numel()], dtype=torch.int64, device="cuda")
        return ops.int_nbit_split_embedding_codegen_lookup_function(
            self.table, self.no_uvm, self.placements, self.weights_offsets, self.weights_tys, self.D_offsets, DIM, 0, DIM, 0, 0, 0, tokens, offsets,
            ops.POOL_NONE, None, ops.BF16, row_alignment=16)

    def project(self, tokens):
        return (self.embed(tokens) @ self.w_qkv).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM)

    def vocabulary(self, attended):
        return (attended.reshape(-1, HEADS * HEAD_DIM) @ self.w_out) @ self.w_vocab

    def take(self, tokens, new_tokens, status):
        """Writes the rows of new tokens into the cache; the projections of all of them."""
        t = decode.kv_block_tables(self.lengths, new_tokens, self.block_tables, self.free_blocks, self.free_start, BLOCK, tokens.numel(), status=status)
        self.lengths, self.free_start = t.lengths, t.free_start
        qkv = self.project(tokens)
        decode.kv_cache_append(qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:], self.key_cache, self.value_cache, t.slots, status=status)
        return qkv, t

    def next_logits(self, query):
        attended, _ = decode.paged_attention(query, self.key_cache, self.value_cache, self.block_tables, self.lengths)
        return self.vocabulary(attended)


def generate(requests=6, steps=24, rows8=False, seed=0):
    """The tokens of every request, prompts in front, and their lengths; the last step's logits before penalties, and the decoder."""
    g = torch.Generator().manual_seed(seed)
    prompt = [1 + int(torch.randint(0, 40, (1,), generator=g)) for _ in range(requests)]
    d = Decoder(requests, max(prompt) + steps, rows8, seed)
    status = ops.Status()
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in prompt]
    lengths = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    # the prompts' rows; the query is each one's last token
    qkv, t = d.take(torch.cat(prompts).cuda(), lengths, status)
    query = qkv[t.offsets[1:].long() - 1, :HEADS]
    one = torch.ones_like(lengths)
    frequency = torch.full((requests,), 0.4, device="cuda")
    # what was said: room for all of it, in lists of equal length whose unsaid end is no token
    said = torch.full((requests, max(prompt) + steps), -1, dtype=torch.int64, device="cuda")
    for r, p in enumerate(prompts):
        said[r, :len(p)] = p.cuda()
    offsets = torch.arange(requests + 1, device="cuda") * said.shape[1]
    for step in range(steps):
        logits = d.next_logits(query)
        ready = decode.penalize_logits(logits, said.view(-1), offsets, lengths.long(), frequency=frequency)
        token = ready.float().argmax(-1)
        said[torch.arange(requests, device="cuda"), d.lengths.long()] = token
        if step < steps - 1:
            qkv, t = d.take(token, one, status)
            query = qkv[:, :HEADS]
    bits, _ = status.read()
    if bits:
        raise RuntimeError(f"a step met an input error: {bits}")
    return said, d.lengths + 1, logits, d


def dense_logits(d, tokens):
    """What the layer gives for one request's tokens behind the last of them, without a cache, in fp32 from the projections on."""
    qkv = d.project(tokens)
    q = qkv[-1, :HEADS].float().view(KV_HEADS, HEADS // KV_HEADS, HEAD_DIM)
    k, v = (x.float().transpose(0, 1).contiguous() for x in (qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]))
    weights = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * HEAD_DIM ** -0.5, -1)
    return d.vocabulary(torch.matmul(weights, v).bfloat16())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--rows8", action="store_true", help="keep keys and values as 8-bit rows")
    a = ap.parse_args()
    said, lengths, logits, d = generate(a.requests, a.steps, a.rows8)
    worst = 0.0
    for r in range(a.requests):
        n = int(lengths[r])
        print("request %d: %s ... %s" % (r, said[r, :4].tolist(), said[r, n - 4:n].tolist()))
        want = dense_logits(d, said[r, :n - 1])
        worst = max(worst, float((logits[r].float() - want.float()).norm() / want.float().norm()))
    print("last step's logits against the dense layer: %.2g relative" % worst)


if __name__ == "__main__":
    main()
