"""Continuous batching over a 4-bit key/value cache: one attention layer of a small
decoder (random weights in 4 bits), requests that arrive, grow and end.

    python3 -m examples.serve [steps]

A step takes any mixture of prompts and single tokens.  On the device, in order:
blocks of ended requests go back (kv_release), the step's block table, slots and
lengths follow from the requests' lengths (kv_plan), the embedding and the fused
projection of the step's tokens (embed_tokens, quantized_matmul), their keys and
values into the cache (kv_append), attention over it (kv_attention), the output
projection and the tied head.  The host knows only lengths and token ids.
"""
import sys

import numpy as np

from cider_press_amd import kernels as K
from cider_press_amd.kernels import embed, kv, qmm
from cider_press_amd.synthetic import from_bits, make_weight

DTYPE = "bf16"


class Server:
    def __init__(self, device, seqs=8, n_blocks=256, block_size=16, max_blocks=32, heads=14, kv_heads=2, dim=64,
                 hidden=896, vocab=2048, seed=0):
        self.device, self.cmds, self.library = device, device.commands(), K.KernelLibrary.quantized(device)
        self.seqs, self.block_size, self.max_blocks = seqs, block_size, max_blocks
        self.heads, self.kv_heads, self.dim, self.hidden, self.vocab = heads, kv_heads, dim, hidden, vocab
        rng = np.random.default_rng(seed)

        def weight(n, k):
            w, s, b = make_weight(rng, n, k, 64, 4, DTYPE)
            return [device.upload(a.reshape(-1), t) for a, t in ((w, "u32"), (s, DTYPE), (b, DTYPE))]

        self.table_w = weight(vocab, hidden)  # the embedding and, tied, the head
        self.qkv_w = weight((heads + 2 * kv_heads) * dim, hidden)
        self.out_w = weight(hidden, heads * dim)
        self.cache = kv.KvCache(device, DTYPE, n_blocks, block_size, kv_heads, dim, 64)
        self.table = self._u32(np.full((seqs, max_blocks), kv.NO_SLOT))
        self.free, self.free_count = self._u32(np.arange(n_blocks)), self._u32([n_blocks])
        self.lens = self._u32(np.zeros(seqs))

    def _u32(self, a):
        return self.device.upload(np.asarray(a, np.uint32).reshape(-1), "u32")

    def step(self, tokens, finished=()):
        """tokens: {request: its new token ids}; finished: requests whose blocks go
        back first (they may take new tokens in the same step).  Returns the logits
        of every request's last token."""
        new = [len(tokens.get(r, ())) for r in range(self.seqs)]
        n, d, cmds = sum(new), self.device, self.cmds
        lens, count, starts, lengths, slots, positions, left = (
            d.alloc_buffer(k, "u32") for k in (self.seqs, 1, self.seqs + 1, self.seqs, n, n, 1))
        shape = (self.table, self.max_blocks, self.block_size)
        kv.kv_release(cmds, self._u32([r in finished for r in range(self.seqs)]), self.lens, *shape, self.free,
                      self.free_count, lens, count)
        kv.kv_plan(cmds, lens, self._u32(new), *shape, self.free, count, starts, lengths, slots, positions, left)

        rows = (self.heads + 2 * self.kv_heads) * self.dim
        x, qkv, a, y, logits = (d.alloc_buffer(n * k, DTYPE) for k in
                                (self.hidden, rows, self.heads * self.dim, self.hidden, self.vocab))
        ids = self._u32(np.concatenate([np.asarray(tokens[r]) for r in sorted(tokens)]))
        embed.embed_tokens(cmds, self.library, *self.table_w, ids, x, self.vocab, self.hidden, 64, 4)
        qmm.quantized_matmul(cmds, *self.qkv_w, x, qkv, n, rows, self.hidden, 64, 4)
        # Queries, keys and values are slices of the fused rows.
        k_at, v_at, strides = self.heads * self.dim, (self.heads + self.kv_heads) * self.dim, (rows, self.dim)
        kv.kv_append(cmds, self.cache, qkv.slice(k_at, len(qkv) - k_at), qkv.slice(v_at, len(qkv) - v_at), slots, n,
                     k_strides=strides, v_strides=strides)
        kv.kv_attention(cmds, self.cache, qkv, self.table, self.max_blocks, starts, lengths, a, n, self.heads, self.seqs,
                        max(new), self.max_blocks * self.block_size, self.dim ** -0.5, q_strides=strides)
        qmm.quantized_matmul(cmds, *self.out_w, a, y, n, self.hidden, self.heads * self.dim, 64, 4)
        qmm.quantized_matmul(cmds, *self.table_w, y, logits, n, self.vocab, self.hidden, 64, 4)
        cmds.commit_and_wait()
        self.lens, self.free_count = lengths, left
        ends = np.cumsum(new)
        out = from_bits(logits.to_numpy(), DTYPE).reshape(n, self.vocab)
        return {r: out[ends[r] - 1] for r in tokens}


def main(steps=12):
    server, rng = Server(K.Device.system_default()), np.random.default_rng(1)
    running, waiting, finished = {}, [int(v) for v in rng.integers(1, 200, 20)], []
    for step in range(steps):
        tokens = {r: ids[-1:] for r, ids in running.items()}
        for r in range(server.seqs):
            if r not in running and waiting and step % 2 == 0:  # a prompt takes the place
                running[r] = rng.integers(0, server.vocab, waiting.pop()).tolist()
                tokens[r] = running[r]
        if not tokens:
            break
        logits = server.step(tokens, finished)
        finished = []
        for r, row in logits.items():
            running[r].append(int(row.argmax()))
            if running[r][-1] % 7 == 0:  # ends here
                finished.append(r)
                print(f"step {step}: request {r} ended with {len(running.pop(r))} tokens")
        print(f"step {step}: {sum(len(t) for t in tokens.values())} tokens of {len(tokens)} requests, "
              f"{int(server.free_count.to_numpy()[0])} blocks free")


if __name__ == "__main__":
    main(*map(int, sys.argv[1:2]))
