"""PagedLM: NanoLLM over prompts of different lengths and a 4-bit paged cache --
the packed prompt attention, the cache, its attention and its page operations
(matrix_ops.attention_packed, kv4) as a serving loop uses them.

    python -m freeml_b200.paged_lm        # a small run on random weights

The forward is NanoLLM's (Examples/NanoLLM/NanoLLM.cpp:268-358) through the
operators of matrix_ops, row by row the one that lm.NanoLM decodes; weights come
in the same packed order.  A sequence lives in a slot of the cache and can be
forked there (several continuations of one prompt share its full pages), freed,
and the cache compacted.  A step or a fork that finds no free page raises and
changes nothing; it can be made again once sequences have been freed.  lm.NanoLM,
with an fp32 cache of equal prompts, is the faster loop (32 sequences, 512 wide, 8
layers: 129,000 tokens/s on a B200, this one 23,000, for its launches from Python);
this one holds 5 bits a value where that holds 32.
"""
from __future__ import annotations

import numpy as np
import torch

from . import kv4, matrix_ops as M
from .lm import NanoLLMShape


class PagedLM:
    def __init__(self, shape: NanoLLMShape, params: torch.Tensor, pages: int, page_size: int = 32, slots: int = 8):
        """params: packed parameters on the device (fp32); pages: of the cache, page_size rows of every layer each."""
        s, d = shape, shape.d_model
        if params.numel() != s.param_count() or not params.is_cuda or params.dtype != torch.float32:
            raise kv4.FmlError(1, "PagedLM", f"expected {s.param_count()} float32 CUDA parameters")
        self.shape, self.hd = shape, d // s.n_head
        at = 0

        def take(*dims):
            nonlocal at
            n = int(np.prod(dims))
            at += n
            return params[at - n:at].view(*dims)

        self.tok, self.pos = take(s.vocab, d), take(s.context, d)
        self.layers = [dict(ln0=take(d), qkv=take(d, 3 * d), proj=take(d, d), ln1=take(d), fc=take(d, 4 * d),
                            mlp=take(4 * d, d)) for _ in range(s.n_layer)]
        self.lnf = take(d)
        self.device = params.device
        self.cache = kv4.KV4Cache(s.n_layer, s.n_head, self.hd, pages, page_size, slots, -(-s.context // page_size),
                                  device=params.device)
        self.length = [0] * slots  # the cache's lens, known to the host
        self.outcome = torch.zeros(1, dtype=torch.int32, device=params.device)  # status word of this class's own calls

    def _ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.device)

    def _slots(self, what, slot_ids, each_once=True):
        """The slots as whole numbers; refused unless they exist (and are named once): the cache would refuse them, or
        take them for others than `length` does."""
        ids = [int(i) for i in slot_ids]
        if any(not 0 <= i < len(self.length) for i in ids) or (each_once and len(set(ids)) != len(ids)):
            raise kv4.FmlError(1, "PagedLM", f"{what}: slots of 0 .. {len(self.length) - 1}"
                                             f"{', each named once' if each_once else ''}")
        return ids

    def _refused(self):
        """Why the page operation just made was refused, or 0 (waits for it)."""
        bits = int(self.outcome.item())
        if bits:
            self.outcome.zero_()
        return bits

    def _forward(self, tokens, positions, counts, slot_ids, prompt: bool):
        """Hidden rows of new tokens (entry b's counts[b] rows in order); their keys and values go into the cache."""
        s, d, T = self.shape, self.shape.d_model, len(tokens)
        new = lambda *dims: torch.empty(*dims, dtype=torch.float32, device=self.device)  # noqa: E731
        starts, ids = self._ints([0] + list(np.cumsum(counts))), self._ints(slot_ids)
        x, where, h, y, qkv, f = new(T, d), new(T, d), new(T, d), new(T, d), new(T, 3 * d), new(T, 4 * d)
        M.GatherRows(x, self.tok, torch.tensor(tokens, dtype=torch.float32, device=self.device))
        M.GatherRows(where, self.pos, torch.tensor(positions, dtype=torch.float32, device=self.device))
        M.Add(x, x, where)
        q, k, v = (qkv.view(T, 3, s.n_head, self.hd)[:, i] for i in range(3))
        att, scale = y.view(T, s.n_head, self.hd), 1.0 / float(np.sqrt(self.hd))
        c = self.cache
        kv4.reserve(c.refs, c.table, c.lens, self._ints(counts), c.page_size, self.outcome, ids)
        bits = self._refused()
        if not bits:
            for slot, n in zip(slot_ids, counts):
                self.length[slot] += n
        elif prompt:  # it reads no cache: check() tells that the slots have stayed empty
            c.status.bitwise_or_(bits)
        else:
            raise kv4.FmlError(5, "PagedLM", "step: " + kv4.reasons(bits))
        for i, w in enumerate(self.layers):
            M.LayerNormOp(h, x, w["ln0"])
            M.Mul(qkv, h, w["qkv"])
            if not bits:
                kv4.append(c.pool[i], c.table, c.lens, k, v, starts, ids)
            if prompt:  # a prompt's rows see each other as they are
                M.attention_packed(att, q, k, v, starts, scale)
            else:
                c.attention(i, att, q, scale, ids)
            M.Mul(h, y, w["proj"], M.RIGHT)
            M.Add(x, x, h)
            M.LayerNormOp(h, x, w["ln1"])
            M.Mul(f, h, w["fc"])
            M.GeluMat(f, f)
            M.Mul(h, f, w["mlp"])
            M.Add(x, x, h)
        return x

    def _logits(self, rows):
        h = torch.empty_like(rows)
        M.LayerNormOp(h, rows, self.lnf)
        out = torch.empty(rows.shape[0], self.shape.vocab, dtype=torch.float32, device=self.device)
        M.Mul(out, h, self.tok, M.RIGHT)
        return out

    def prefill(self, prompts, slot_ids):
        """Run prompts (lists of token ids, of any lengths) into empty slots; the logits after each one's last row.
        Where the pages do not suffice all of the slots stay empty, which cache.check() tells (the logits are right)."""
        counts, slot_ids = [len(p) for p in prompts], self._slots("prefill", slot_ids)
        if any(n < 1 or n > self.shape.context for n in counts) or any(self.length[i] for i in slot_ids) \
                or len(slot_ids) != len(counts):
            raise kv4.FmlError(1, "PagedLM", "prefill: prompts of 1 .. context tokens, one empty slot each")
        tokens = [int(t) for p in prompts for t in p]
        x = self._forward(tokens, [i for n in counts for i in range(n)], counts, slot_ids, prompt=True)
        return self._logits(x[(torch.tensor(np.cumsum(counts), device=self.device) - 1)].contiguous())

    def step(self, tokens, slot_ids):
        """One more token of each slot; the logits after it.  Raises, with nothing changed, where a page is missing."""
        slot_ids = self._slots("step", slot_ids)
        positions = [self.length[i] for i in slot_ids]
        if len(tokens) != len(slot_ids):
            raise kv4.FmlError(1, "PagedLM", f"step: {len(tokens)} tokens, {len(slot_ids)} slots")
        if any(p < 1 or p >= self.shape.context for p in positions):
            raise kv4.FmlError(1, "PagedLM", "step: a slot that is empty, or whose context is full")
        return self._logits(self._forward([int(t) for t in tokens], positions, [1] * len(slot_ids), slot_ids, prompt=False))

    def fork(self, parents, children):
        parents, children = self._slots("fork", parents, False), self._slots("fork", children)
        if len(parents) != len(children) or any(self.length[i] for i in children):
            raise kv4.FmlError(1, "PagedLM", "fork: an empty child for each parent")
        c = self.cache
        kv4.fork(c.pool, c.refs, c.table, c.lens, self._ints(parents), self._ints(children), self.outcome)
        bits = self._refused()
        if bits:
            raise kv4.FmlError(5, "PagedLM", "fork: " + kv4.reasons(bits))
        for parent, child in zip(parents, children):
            self.length[child] = self.length[parent]

    def free(self, slot_ids):
        slot_ids = self._slots("free", slot_ids, False)
        self.cache.free(self._ints(slot_ids))
        for i in slot_ids:
            self.length[i] = 0

    def compact(self):
        self.cache.compact()


def main():
    from .lm import CONFIGS, prompt_tokens, random_params
    shape = CONFIGS[1]["shape"]
    lm = PagedLM(shape, random_params(shape, 0), pages=24, page_size=16, slots=6)
    prompts = [prompt_tokens(seed, shape.vocab, 1, n)[0] for seed, n in ((1, 16), (2, 41), (3, 7))]
    logits = lm.prefill(prompts, [0, 1, 2])
    # the second prompt's two likeliest continuations go on side by side
    best = logits[1].topk(2).indices.tolist()
    lm.fork([1], [3])
    slots, tokens = [0, 1, 2, 3], [int(logits[0].argmax()), best[0], int(logits[2].argmax()), best[1]]
    written = {i: [t] for i, t in zip(slots, tokens)}
    for _ in range(24):
        tokens = lm.step(tokens, slots).argmax(-1).tolist()
        for i, t in zip(slots, tokens):
            written[i].append(t)
    for i in slots:
        print(f"slot {i}: {lm.length[i]} rows, continued with {written[i]}")
    lm.free([0, 1])
    lm.compact()
    lm.cache.check()
    used = int((lm.cache.refs > 0).sum())
    values = 2 * shape.n_layer * shape.d_model
    print(f"after two sequences ended: {used} of {lm.cache.refs.numel()} pages, all at the front; "
          f"{lm.cache.pool.numel() / (lm.cache.refs.numel() * lm.cache.page_size):.0f} bytes a row of all layers, {4 * values} in fp32")


if __name__ == "__main__":
    main()
