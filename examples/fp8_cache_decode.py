"""A layer's serving loop over a key/value cache held in 8 bits: prompts of different lengths in one batch, then single tokens.

Each step takes the packed projection of its new tokens, appends their rotated keys and values to the cache and attends over it:

    PagedKvAppendFp8     rotates queries and keys, finds the blocks' scales, writes the codes
    PagedAttentionFp8    new tokens' queries over all that their sequences have in the cache

Here the projections are random numbers.  The results are compared with attention in 32 bits over keys and values that were never
rounded to 8 bits.  Run: python examples/fp8_cache_decode.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer  # noqa: E402

HEADS, KV_HEADS, DIM, BLOCK = 16, 4, 128, 16
PROMPTS, STEPS = [300, 17, 129], 8


def rotate(x, cos, sin):
    """Pairs (2i, 2i + 1) of x [tokens, heads, DIM] by cos, sin [tokens, DIM / 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def main():
    torch.manual_seed(0)
    backend, batch, longest = CudaBackend(), len(PROMPTS), max(PROMPTS) + STEPS
    columns = -(-longest // BLOCK)
    cache = backend.AllocateKvCacheFp8(batch * columns, BLOCK, KV_HEADS, DIM)
    tables = GpuBuffer(torch.randperm(batch * columns).to(torch.int32).cuda())   # the blocks of a sequence lie anywhere
    angle = torch.arange(longest)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2) / DIM)
    cos, sin = GpuBuffer(angle.cos().float().cuda()), GpuBuffer(angle.sin().float().cuda())

    lens, new = [0] * batch, PROMPTS
    keys, values = [[] for _ in PROMPTS], [[] for _ in PROMPTS]   # in 32 bits, for the comparison
    worst = 0.0
    for step in range(1 + STEPS):
        tokens, starts = sum(new), [0]
        for n in new:
            starts.append(starts[-1] + n)
        qkv = torch.randn(tokens, HEADS + 2 * KV_HEADS, DIM, device="cuda").bfloat16()
        queries, out = (GpuBuffer(torch.empty(tokens, HEADS, DIM, dtype=torch.bfloat16, device="cuda")) for _ in range(2))
        first = GpuBuffer(torch.tensor(starts, dtype=torch.int32, device="cuda"))
        before = GpuBuffer(torch.tensor(lens, dtype=torch.int32, device="cuda"))
        lens_now = [a + n for a, n in zip(lens, new)]
        after = GpuBuffer(torch.tensor(lens_now, dtype=torch.int32, device="cuda"))

        backend.PagedKvAppendFp8(GpuBuffer(qkv), queries, cache, tables, before, batch, tokens, HEADS, columns, cos=cos, sin=sin,
                                 tokenStarts=first)
        backend.PagedAttentionFp8(queries, cache, tables, after, out, batch, HEADS, max(new), max(lens_now), columns, DIM ** -0.5,
                                  queryStarts=first)

        for b in range(batch):
            rows, at = slice(starts[b], starts[b + 1]), slice(lens[b], lens_now[b])
            q, k, v = qkv[rows].float().split((HEADS, KV_HEADS, KV_HEADS), 1)
            q = rotate(q, cos.tensor[at], sin.tensor[at])
            keys[b].append(rotate(k, cos.tensor[at], sin.tensor[at]))
            values[b].append(v)
            k, v = (torch.cat(x[b]).repeat_interleave(HEADS // KV_HEADS, 1) for x in (keys, values))
            seen = torch.arange(lens_now[b], device="cuda") <= torch.arange(lens[b], lens_now[b], device="cuda")[:, None]
            s = torch.einsum("ihd,jhd->hij", q, k) * DIM ** -0.5
            p = s.masked_fill(~seen, float("-inf")).softmax(-1)
            ref = torch.einsum("hij,jhd->ihd", p, v)
            worst = max(worst, ((out.tensor[rows].float() - ref).norm() / ref.norm()).item())
        lens, new = lens_now, [1] * batch
    held = cache.keys.SizeInBytes + cache.values.SizeInBytes + cache.keyScales.SizeInBytes + cache.valueScales.SizeInBytes
    print(f"{1 + STEPS} steps, {sum(lens)} tokens, cache of {held >> 10} KB; relative error by the 8 bits at most {worst:.3f}")
    assert worst < 0.08, worst


if __name__ == "__main__":
    main()
