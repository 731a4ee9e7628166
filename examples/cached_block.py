"""Transformer blocks that serve: packed linears, the norms between them, a paged 8-bit cache of keys and values and attention over it.

    python examples/cached_block.py

A prompt goes through a few blocks at once; the sequence is forked (a beam, or the two sides of a guided step), both go on token by
token, one ends, and the pool is compacted. Every step is the library's own calls on one stream; nothing waits for the device
in between. At the end the last token is computed once more from the whole sequence at once, and both ways are compared.
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from __graft_entry__ import load_package  # noqa: E402

WIDTH, HEADS, KV_HEADS, HEAD_DIM, MLP, LAYERS = 1024, 8, 2, 128, 2048, 3
PAGE, PAGES, SEQUENCES, LONGEST = 32, 64, 4, 512
QKV = (HEADS + 2 * KV_HEADS) * HEAD_DIM


def ok(status):
    if status != 0:
        raise RuntimeError(f"cuda status {status}")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Model:
    """Random packed weights. All linears take 16-bit activations: with 4-bit ones both ways at the end would be a tenth apart, since a
    difference of half a percent, as 8-bit keys and values give it, moves one code of a hundred by a step of two fifths of a deviation."""

    def __init__(self, qi, seed=7):
        self.qi, self.random = qi, torch.Generator(device="cuda").manual_seed(seed)
        self.layers = [{"norm1": self.uniform(WIDTH), "norm2": self.uniform(WIDTH), "qkv": self.record(qi.SCHEME_W4A16, QKV, WIDTH), "out": self.record(qi.SCHEME_W4A16, WIDTH, HEADS * HEAD_DIM),
                        "fc1": self.record(qi.SCHEME_W4A16, MLP, WIDTH), "fc2": self.record(qi.SCHEME_W4A16, WIDTH, MLP)} for _ in range(LAYERS)]
        self.last_norm = self.uniform(WIDTH)

    def uniform(self, n):
        return torch.rand(n, device="cuda", generator=self.random) + 0.5

    def record(self, scheme, n, k):
        """Codes of a bell shape whose values have deviation 0.03."""
        codes = (torch.randn(n, k, device="cuda", generator=self.random) * 3 + 7.5).round().clamp(0, 15).to(torch.uint8)
        scales = torch.full((n, k // 64), 0.01, device="cuda", dtype=torch.float16)
        return self.qi.PackedLinear(scheme, n, k, (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales, (scales * -7.5).half())


class Server:
    """The cache, its pages and the buffers that the blocks work in."""

    def __init__(self, qi, model):
        self.qi, self.model = qi, model
        shape, scales = (LAYERS, PAGES, KV_HEADS, PAGE, HEAD_DIM), (LAYERS, PAGES, KV_HEADS, PAGE // qi.KV_BLOCK)
        byte = dict(dtype=torch.uint8, device="cuda")
        self.cache = qi.KvCache(torch.empty(*shape, **byte), torch.empty(*shape, **byte), torch.empty(*scales, device="cuda"), torch.empty(*scales, device="cuda"))
        self.pages = qi.KvPages(torch.full((SEQUENCES, -(-LONGEST // PAGE)), -1, dtype=torch.int32, device="cuda"), ints([0] * SEQUENCES), ints([0] * PAGES))
        self.page_work = torch.empty(qi.kv_pages_workspace(self.cache, self.pages), **byte)
        self.words, self.used, self.room = [], ints([0]), None  # what reservations and forks told, a word each: nothing waits for it
        most = qi.KvBatch(None, ints([0] * (SEQUENCES + 1)), SEQUENCES * LONGEST, LONGEST)  # no step is larger
        self.attention_work = torch.zeros(qi.kv_attention_workspace(self.cache, most, HEADS, LONGEST), **byte)
        self.work = qi.LinearWork(torch.empty(LONGEST, MLP // 2, **byte), torch.empty(LONGEST, MLP // 64, dtype=torch.float16, device="cuda"),
                                  torch.empty(LONGEST, MLP, dtype=torch.float16, device="cuda"), torch.empty(LONGEST, MLP, **byte))

    def word(self):
        self.words.append(ints([0]))
        return self.words[-1]

    def reserve(self, slots, counts):
        self.room = self.word()  # forward() leaves the cache alone where there is none
        ok(self.qi.kv_pages_reserve_ex(self.cache, self.pages, ints(slots), ints(counts), len(slots), self.room, self.page_work))

    def fork(self, parent, child):
        ok(self.qi.kv_pages_fork_ex(self.cache, self.pages, ints([parent]), ints([child]), 1, self.word(), self.page_work))

    def end(self, slot):
        ok(self.qi.kv_pages_free_ex(self.cache, self.pages, ints([slot]), 1))

    def compact(self):
        ok(self.qi.kv_pages_compact_ex(self.cache, self.pages, self.used, self.page_work))

    def forward(self, slots, counts, tokens):
        """The hidden states of `tokens` [sum(counts), WIDTH], which are the last counts[i] tokens of sequence slots[i]."""
        qi, rows = self.qi, sum(counts)
        half = dict(dtype=torch.float16, device="cuda")
        batch = qi.KvBatch(ints(slots), ints([sum(counts[:i]) for i in range(len(counts) + 1)]), rows, max(counts), self.room)
        residual, x = tokens.clone(), torch.empty(rows, WIDTH, **half)
        qkv, y, out, hidden = torch.empty(rows, QKV, **half), torch.empty(rows, HEADS * HEAD_DIM, **half), torch.empty(rows, WIDTH, **half), torch.empty(rows, MLP, **half)

        def norm(weight, branch):
            ok(qi.gated_norm_ex(qi.GatedNorm(rows, WIDTH, kind=qi.NORM_RMS, residual=residual, branch=branch, branch_dtype=qi.DTYPE_F16, residual_out=residual, weight=weight, y=x,
                                             y_dtype=qi.DTYPE_F16)))

        def linear(record, source, to):
            ok(qi.linear(record, self.work, source, to, rows, input_dtype=qi.DTYPE_F16, output_dtype=qi.DTYPE_F16))

        branch = None
        for i, layer in enumerate(self.model.layers):
            norm(layer["norm1"], branch)
            linear(layer["qkv"], x, qkv)
            ok(qi.kv_append_ex(self.cache, self.pages, batch, i, qkv[:, HEADS * HEAD_DIM:], qkv[:, (HEADS + KV_HEADS) * HEAD_DIM:], qi.DTYPE_F16, QKV, QKV))
            ok(qi.kv_attention_ex(self.cache, self.pages, batch, i, qkv, QKV, y, HEADS * HEAD_DIM, HEADS, HEAD_DIM ** -0.5, LONGEST, workspace=self.attention_work))
            linear(layer["out"], y, out)
            norm(layer["norm2"], out)
            linear(layer["fc1"], x, hidden)
            linear(layer["fc2"], torch.nn.functional.gelu(hidden, approximate="tanh"), out)
            branch = out
        norm(self.model.last_norm, branch)
        return x


def main():
    qi = load_package()
    model = Model(qi)
    server, g = Server(qi, model), torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randn(140, WIDTH, device="cuda", generator=g)
    prompt, steps = 117, 12
    server.reserve([0], [prompt])
    server.forward([0], [prompt], tokens[:prompt])
    server.fork(0, 2)  # shares the prompt's whole pages
    for i in range(steps):  # both go on, each with a token of its own
        server.reserve([0, 2], [1, 1])
        stepwise = server.forward([0, 2], [1, 1], torch.stack([tokens[prompt + i], -tokens[prompt + i]]))
    server.end(2)
    server.compact()
    server.reserve([0], [1])
    last = server.forward([0], [1], tokens[prompt + steps:prompt + steps + 1])
    # the same sequence at once, in a slot of its own
    count = prompt + steps + 1
    server.reserve([1], [count])
    at_once = server.forward([1], [count], tokens[:count])[-1:]
    torch.cuda.synchronize()
    if qi.kernel_status() != 0 or any(word.item() != 0 for word in server.words):
        raise RuntimeError("a call found something unsound, or no room")
    difference = ((last - at_once).float().norm() / at_once.float().norm()).item()
    print(f"{LAYERS} blocks, {count} tokens: {server.pages.lengths.tolist()} tokens held, {int((server.pages.references > 0).sum())} pages in use, "
          f"step by step against at once: {difference:.1e} apart")
    return difference, stepwise


if __name__ == "__main__":
    main()
