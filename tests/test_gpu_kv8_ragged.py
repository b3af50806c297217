"""Attention over an 8-bit pool where its kernels meet: ragged batches whose sequences are divided between them, long sequences
whose parts are many, numbers of KV heads that do not fill a CTA, capped logits of every size.

Against the formula in 64 bits, with the tolerances of the other tests of this cache; a capped logit is off by another
2^-20 of the cap (tanh is formed to 7e-7 of itself or better)."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_kv8 import Pool, attend, attend64, bounds, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,block", [("bf16", 128, 16), ("f16", 64, 32)])
def test_few_and_many_rows_in_a_batch(dtype, dim, block):
    """Four rows a query: 8 queries are the most of the kernel for few, 9 the fewest of the other; 32 and 33 make one row tile and two."""
    counts = [9, 1, 8, 0, 40, 32, 1, 33, 7, 64, 65]
    lens = [9, 1000, 8, 70, 300, 640, 0, 33, 1, 129, 2100]
    pool = Pool(lens, block, 2, dim, seed=21).cuda()
    check(pool, queries(sum(counts), 8, dim, dtype, 22), lens, counts, 8, dtype=dtype)


def test_only_few_rows_where_more_were_allowed():
    counts, lens = [1, 2, 1], [400, 90, 33]
    pool = Pool(lens, 16, 2, 128, seed=23).cuda()
    check(pool, queries(4, 8, 128, "bf16", 24), lens, counts, 8, dtype="bf16", uniform=False, max_q=200)


def test_only_many_rows_in_a_ragged_batch():
    counts, lens = [100, 130, 90], [400, 130, 333]
    pool = Pool(lens, 16, 2, 128, seed=25).cuda()
    check(pool, queries(320, 8, 128, "bf16", 26), lens, counts, 8, dtype="bf16", uniform=False)


def test_more_query_heads_a_group_than_few_rows():
    """64 query heads to a KV head: no sequence has few rows."""
    counts, lens = [1, 3, 1], [400, 90, 33]
    pool = Pool(lens, 16, 1, 64, seed=27).cuda()
    check(pool, queries(5, 64, 64, "f16", 28), lens, counts, 64, dtype="f16", uniform=False)


@pytest.mark.parametrize("kv_heads", [1, 2, 3, 5, 6, 8, 16])
@pytest.mark.parametrize("count", [1, 3])
@pytest.mark.parametrize("block", [16, 24])
def test_numbers_of_kv_heads(kv_heads, count, block):
    """Warps of a CTA that go through 1, 2, 4 or 8 heads side by side; 5 rows a group and query."""
    lens = [500, 61, 1200]
    pool = Pool(lens, block, kv_heads, 64, seed=29).cuda()
    check(pool, queries(3 * count, 5 * kv_heads, 64, "bf16", 30), lens, [count] * 3, 5 * kv_heads, dtype="bf16")


@pytest.mark.parametrize("kv_heads,dtype", [(1, "bf16"), (4, "f16"), (2, "f32")])
def test_long_sequence_of_many_parts(kv_heads, dtype):
    """20000 keys of one sequence beside short ones: a line in over a hundred parts, blocks beyond a lane's first 64."""
    lens = [20000, 5, 130]
    pool = Pool(lens, 16, kv_heads, 64, seed=31).cuda()
    check(pool, queries(3, 2 * kv_heads, 64, dtype, 32), lens, [1] * 3, 2 * kv_heads, dtype=dtype)


def test_tiny_blocks():
    """A tile of keys in sixteen blocks."""
    lens = [700, 33]
    pool = Pool(lens, 1, 2, 64, seed=33).cuda()
    check(pool, queries(2, 4, 64, "bf16", 34), lens, [1, 1], 4, dtype="bf16")


@pytest.mark.parametrize("count", [1, 2])
def test_hundreds_of_sequences(count):
    """More sequences than lanes, some without keys."""
    g = np.random.default_rng(35)
    lens = [int(n) for n in g.integers(0, 90, 300)]
    pool = Pool(lens, 16, 2, 64, seed=36).cuda()
    check(pool, queries(300 * count, 4, 64, "bf16", 37), lens, [count] * 300, 4, dtype="bf16")


@pytest.mark.parametrize("factor", [0.05, 0.5, 4.0, 100.0])
@pytest.mark.parametrize("counts", [[1, 1], [150, 60]])
@pytest.mark.parametrize("dim", [64, 128])
def test_softcap_of_small_and_large_logits(factor, counts, dim):
    """Logits far below the cap, around it and far above."""
    lens, cap, scale = [900, 77], 7.0, 1 / math.sqrt(dim)
    pool = Pool(lens, 16, 2, dim, seed=38).cuda()
    q = queries(sum(counts), 8, dim, "bf16", 39) * factor
    o, lse, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, 8, scale=scale, softcap=cap)
    # (a product of 32 bits that is off by e is off by no more behind the cap)
    bo, bl = bounds(o, lse, a, top, "bf16", "bf16", dim)
    bo, bl = bo + 2.1 * 2.0 ** -20 * cap * a, bl + 2.0 ** -20 * cap
    go, gl = attend(pool, q, lens, counts, 8, dtype="bf16", softcap=cap)
    assert (np.abs(go.double().cpu().numpy() - o) <= bo).all()
    assert (np.abs(gl.double().cpu().numpy() - lse) <= bl).all()


def test_results_do_not_depend_on_what_else_runs():
    """The same call again and again, alone and beside others: bit for bit the same."""
    counts, lens = [1, 9, 2, 70], [3000, 900, 1400, 600]
    pool = Pool(lens, 16, 2, 128, seed=40).cuda()
    q = queries(sum(counts), 8, 128, "bf16", 41)
    first = attend(pool, q, lens, counts, 8, dtype="bf16")
    other = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(other):
            attend(pool, q, lens, counts, 8, dtype="bf16", stream=other.cuda_stream, poll=False)
        again = attend(pool, q, lens, counts, 8, dtype="bf16")
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    torch.cuda.synchronize()


@pytest.mark.parametrize("dim", [16, 32, 48, 80, 112, 144, 208, 240])
@pytest.mark.parametrize("dtype,count", [("bf16", 1), ("f16", 6), ("f32", 1), ("f32", 4)])
def test_head_sizes_between_the_tiles(dim, dtype, count):
    """Head sizes that fill a part of a kernel's 64, 128 or 256 columns; blocks of 16 and of 40 tokens."""
    for block, lens in ((16, [300, 77]), (40, [33, 410])):
        pool = Pool(lens, block, 2, dim, seed=42).cuda()
        check(pool, queries(2 * count, 6, dim, dtype, 43), lens, [count] * 2, 6, dtype=dtype)
