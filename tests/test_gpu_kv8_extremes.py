"""Attention over an 8-bit pool far from ordinary values: large logits, NaN, scales far apart."""
import math

import numpy as np
import pytest
import torch

from aidotnet.tensors_b200 import native as N
from tests._harness import TORCH_DT
from tests.test_gpu_kv8 import Pool, attend, attend64, bounds, queries

pytestmark = pytest.mark.gpu

CODES = {0: (0x38, 0x3c, 0x3e), 1: (0x30, 0x34, 0x36)}   # 1, 1.5, 1.75, and half of each


def tied(lens, block, kv_heads, dim, seed):
    """A pool whose keys begin with 2^-7 times 1, 1.5 or 1.75, in blocks of two scales: many keys share the largest logit of a query
    that looks at the first element alone, exactly, and the next one is far below."""
    pool = Pool(lens, block, kv_heads, dim, seed=seed)
    g = np.random.default_rng(seed)
    half = g.integers(0, 2, pool.scales[0].shape)
    pick = g.integers(0, 3, pool.codes[0].shape[:3])
    table = np.array([CODES[0], CODES[1]], np.uint8)
    pool.codes[0][..., 0] = table[half[:, None, :], pick]
    pool.scales[0] = np.exp2(half - 7.0).astype(np.float32)
    return pool.cuda()


def looking_at_the_first(n, heads, dim, dtype, sign):
    q = torch.zeros((n, heads, dim))
    q[..., 0] = sign
    return q.to(TORCH_DT[dtype]).cuda()


def check_tied(lens, counts, heads, kv_heads, dim, block, dtype, exponent, sign, out=None, **kw):
    """A query's logits to base 2 are about 2^exponent.  Equal logits are equal in 32 bits too (the scales are powers of two), whatever a
    rounding of 2^(exponent - 24) does to them, so that the weights of those that share the maximum are equal to 2^-11 and all others are zero."""
    pool = tied(lens, block, kv_heads, dim, seed=50 + exponent)
    q = looking_at_the_first(sum(counts), heads, dim, dtype, sign)
    scale = 2.0 ** (exponent + 7) / math.log2(math.e)
    o, lse, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, heads, scale=np.float64(np.float32(scale)))
    bo, bl = bounds(o, lse, a, np.zeros_like(top), dtype, out or dtype, dim)
    got, stats = attend(pool, q, lens, counts, heads, dtype=dtype, out=out, scale=scale, **kw)
    got, stats = got.double().cpu().numpy(), stats.double().cpu().numpy()
    assert np.isfinite(got).all() and np.isfinite(stats).all()
    assert (np.abs(got - o) <= bo).all()
    assert (np.abs(stats - lse) <= bl).all()


LARGE = [16, 19, 20, 21, 24, 25, 26, 27, 28, 29, 30, 33, 40, 60]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", LARGE)
@pytest.mark.parametrize("dtype,dim,workspace", [("bf16", 128, True), ("f16", 64, True), ("bf16", 64, False)])
def test_large_logits_of_many_queries(exponent, sign, dtype, dim, workspace):
    check_tied([300, 1290], [150, 70], 8, 2, dim, 16, dtype, exponent, sign, workspace=workspace)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", LARGE)
@pytest.mark.parametrize("dtype,out,dim,count,block", [("bf16", "bf16", 128, 1, 16), ("f16", "f16", 64, 4, 16), ("bf16", "f32", 128, 1, 16), ("f32", "f32", 256, 3, 24)])
def test_large_logits_of_few_queries(exponent, sign, dtype, out, dim, count, block):
    check_tied([300, 1290, 17], [count] * 3, 8, 2, dim, block, dtype, exponent, sign, out=out)


@pytest.mark.parametrize("exponent", [26, 27, 28, 30])
@pytest.mark.parametrize("path", [N.PATH_AUTO, N.PATH_GENERIC])
def test_large_logits_one_after_the_other(exponent, path):
    """Keys whose logits rise by one or two units in the last place of the largest: each new maximum is a little above the one before.  (Within a few
    units the weights depend on how the products were rounded: results lie between the values.)"""
    dim, lens = 64, [900, 333]
    pool = Pool(lens, 16, 2, dim, seed=57)
    pool.codes[0][..., 0], pool.codes[0][..., 1:] = 0x38, 0x38
    pool.scales[0][:] = 1.0
    for b in range(2):
        for j in range(-(-lens[b] // 16)):
            pool.scales[0][pool.table[b, j]] = 1 + j * 2.0 ** -23
    pool.cuda()
    q = looking_at_the_first(2, 4, dim, "bf16", 1)
    out, stats = attend(pool, q, lens, [1, 1], 4, dtype="bf16", scale=2.0 ** exponent / math.log2(math.e), path=path)
    most = max(np.abs(pool.rows(1, b, n)).max() for b, n in enumerate(lens))
    assert bool(out.isfinite().all()) and bool(stats.isfinite().all())
    assert float(out.abs().max()) <= most * (1 + 2.0 ** -7)


@pytest.mark.parametrize("size", [3e2, 2e4, 1e6, 1e12])
@pytest.mark.parametrize("softcap", [0.0, 1e9])
def test_queries_of_a_diverged_model(size, softcap):
    """Normal queries and keys, of logits that differ by far more than a weight can show: results are within the values that they are made of."""
    lens, counts = [700, 900], [400, 128]
    pool = Pool(lens, 16, 2, 128, seed=51).cuda()
    q = queries(sum(counts), 8, 128, "bf16", 52) * size
    out, stats = attend(pool, q, lens, counts, 8, dtype="bf16", softcap=softcap)
    most = max(np.abs(pool.rows(1, b, n)).max() for b, n in enumerate(lens))
    assert bool(out.isfinite().all()) and bool(stats.isfinite().all())
    assert float(out.abs().max()) <= most * (1 + 2.0 ** -7)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("lens,counts,heads", [([300], [90], 2), ([300], [90], 8), ([463], [300], 1), ([100], [100], 4), ([333], [8], 4), ([129], [3], 6)])
def test_nan_anywhere_in_the_last_tiles(lens, counts, heads, which, causal):
    """One NaN among a key's elements or a key's values, at every eighth of the last keys in turn (and at both ends): the rows that see it
    are NaN, the others what they are without it."""
    n, c = lens[0], counts[0]
    pool = Pool(lens, 16, 1, 64, seed=53).cuda()
    q = queries(c, heads, 64, "bf16", 54)
    clean, _ = attend(pool, q, lens, counts, heads, dtype="bf16", causal=causal)
    codes, stash = pool.t[which], pool.t[which].clone()
    for key in sorted({n - 1, *range(max(0, n - 330), n, 8)}):
        at = (int(pool.table[0, key // 16]), key % 16, 0, key % 64)
        codes[at] = 0xff if key % 16 else 0x7f
        dirty, _ = attend(pool, q, lens, counts, heads, dtype="bf16", causal=causal)
        codes[at] = stash[at]
        first = max(0, key - (n - c)) if causal else 0
        nan = dirty.isnan().any(-1).any(-1)
        assert not bool(nan[:first].any()), key
        assert bool(dirty[first:].isnan().any(-1).all()), key
        assert torch.equal(dirty[:first], clean[:first]), key


@pytest.mark.parametrize("factor", [0.02, 20.0])
@pytest.mark.parametrize("which", ["key", "query"])
@pytest.mark.parametrize("dtype,out,counts", [("bf16", "bf16", [1, 1]), ("f16", "f16", [3, 3]), ("f32", "f32", [2, 2]), ("bf16", "f32", [5, 4]), ("bf16", "bf16", [150, 60])])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_behind_a_softcap(dtype, out, counts, which, factor, dim):
    """A NaN key or query element with capped logits, the other logits far below the cap or beyond it: the rows that have it are NaN, no other row is."""
    lens, heads, cap = [400, 100], 8, 5.0
    pool = Pool(lens, 16, 2, dim, seed=55).cuda()
    q = queries(sum(counts), heads, dim, dtype, 56) * factor
    clean, _ = attend(pool, q, lens, counts, heads, dtype=dtype, out=out, softcap=cap)
    hit = torch.zeros(clean.shape[:2], dtype=torch.bool, device="cuda")
    if which == "key":
        key = lens[0] - counts[0] + counts[0] // 2
        pool.t[0][int(pool.table[0, key // 16]), key % 16, 1, 9] = 0x7f
        hit[counts[0] // 2:counts[0], 4:] = True
    else:
        q[counts[0] // 2, 3, 11] = float("nan")
        hit[counts[0] // 2, 3] = True
    dirty, stats = attend(pool, q, lens, counts, heads, dtype=dtype, out=out, softcap=cap)
    assert torch.equal(dirty.isnan().any(-1), hit) and torch.equal(stats.isnan(), hit)
    assert bool(clean.isfinite().all())


def loud_and_quiet(lens, block, dim, seed, loud, quiet, every):
    """Blocks with number 2 mod `every` of a sequence: values of scale 2^loud, and keys whose logits for a query that begins with 60 are about 40 (natural) below those of
    the others, whose values' scale is 2^quiet.  Other elements are ordinary."""
    pool = Pool(lens, block, 2, dim, seed=seed)
    pool.scales[0][:] = 2.0 ** -7
    pool.codes[0][..., 0] = 0
    pool.scales[1][:] = 2.0 ** quiet
    for b in range(pool.batch):
        for j in range(2, -(-lens[b] // block), every):
            pool.codes[0][pool.table[b, j], ..., 0] = 0xfe   # -448
            pool.scales[1][pool.table[b, j]] = 2.0 ** loud
    return pool


VALUE_CASES = [("bf16", "bf16", 128, [1, 1], 16), ("f16", "f16", 64, [4, 4], 16), ("f16", "f32", 64, [1, 1], 24), ("f32", "f32", 64, [5, 3], 16),
               ("bf16", "bf16", 128, [150, 60], 16), ("f16", "f16", 64, [150, 60], 16)]


@pytest.mark.parametrize("dtype,out,dim,counts,block", VALUE_CASES)
@pytest.mark.parametrize("loud,quiet", [(18, -6), (28, -6), (20, -26), (5, -100), (-100, 5), (100, 60)])
def test_large_values_that_have_no_weight(dtype, out, dim, counts, block, loud, quiet):
    """The weights' precision goes by what they add to the result: blocks of large values but weights of 2^-58 cost the others nothing."""
    lens = [700, 410]
    pool = loud_and_quiet(lens, block, dim, 58, loud, quiet, 4)
    if quiet == -100:
        pool.codes[1][:] = np.where((pool.scales[1] == 2.0 ** quiet)[:, None, :, None], 0, pool.codes[1])   # as an append writes zeros
    pool.cuda()
    q = queries(sum(counts), 8, dim, dtype, 59)
    q[..., 0] = 60 * math.sqrt(dim) / math.sqrt(32)
    o, lse, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, 8, scale=1 / math.sqrt(dim))
    bo, bl = bounds(o, lse, a, top, dtype, out, dim)
    got, stats = attend(pool, q, lens, counts, 8, dtype=dtype, out=out)
    got, stats = got.double().cpu().numpy(), stats.double().cpu().numpy()
    if out == "f16":   # (what 16 bits hold)
        assert np.abs(o).max() < 65504 or loud > 30
        o, bo = np.clip(o, -65504, 65504), np.where(np.abs(o) + bo > 65504, np.inf, bo)
    assert (np.abs(got - o) <= bo)[np.isfinite(bo)].all()
    assert (np.abs(stats - lse) <= bl).all()


@pytest.mark.parametrize("dtype,out,dim,counts,block", VALUE_CASES)
@pytest.mark.parametrize("scale", [2.0 ** 30, float("nan"), float("inf")])
def test_scales_of_values_that_a_query_does_not_see(dtype, out, dim, counts, block, scale):
    """Causal: the last block's values have a scale far above the others', or one that is no number.  Queries before that block's first key have the results
    that they have without it, up to how the sums are ordered; those that see it are not finite where it is not."""
    lens = [64 * 5 + 3, 64 * 2 + 2]
    counts = [max(counts[0], 5), max(counts[1], 4)]
    pool = Pool(lens, block, 2, dim, seed=60).cuda()
    q = queries(sum(counts), 8, dim, dtype, 61)
    for b, n in enumerate(lens):
        pool.s[1][int(pool.table[b, (n - 1) // block])] = scale
        pool.scales[1][pool.table[b, (n - 1) // block]] = scale
    with np.errstate(invalid="ignore", over="ignore"):
        o, lse, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, 8, scale=1 / math.sqrt(dim))
    bo, _ = bounds(o, lse, a, top, dtype, out, dim)
    got, _ = attend(pool, q, lens, counts, 8, dtype=dtype, out=out)
    got, r = got.double().cpu().numpy(), 0
    for n, c in zip(lens, counts):
        edge = (n - 1) // block * block   # the block's first key
        blind = max(0, edge - (n - c))    # queries that do not see it
        assert (np.abs(got - o) <= bo)[r:r + blind].all()
        if not math.isfinite(scale):
            assert not np.isfinite(got[r + blind:r + c]).all(-1).any()
        r += c


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", [99, 100, 112, 120])
@pytest.mark.parametrize("dtype,dim,count", [("bf16", 128, 1), ("f32", 64, 3), ("bf16", 128, 150), ("f16", 64, 90)])
def test_logits_of_every_finite_size(exponent, sign, dtype, dim, count):
    """Logits of up to 2^121, none of them above -2^98 where they are negative: the largest still has the weight."""
    check_tied([300, 290], [count] * 2, 8, 2, dim, 16, dtype, exponent, sign)


@pytest.mark.parametrize("kind", [N.MASK_NONE, N.MASK_KEEP_U8, N.MASK_KEEP_F32, N.MASK_ADD_F32])
def test_arrays_between_their_elements_are_refused(kind):
    """Before anything is launched; a mask of bytes may lie anywhere."""
    pool = Pool([40], 16, 2, 64, seed=62).cuda()
    q, out = queries(1, 4, 64, "bf16", 63), torch.empty(4 * 64, dtype=torch.bfloat16, device="cuda")
    lens, starts = torch.tensor([40, 0], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda")
    lse, mask = torch.empty(8, device="cuda"), torch.ones(256, device="cuda")
    h = N.Handle(device=0, qkv_dtype=N.BF16, out_dtype=N.BF16, head_dim=64, num_q_heads=4, num_kv_heads=2, causal=True, emit_lse=True, mask_kind=kind)
    good = dict(q=q.data_ptr(), out=out.data_ptr(), cache=pool.packed(), batch=1, seq_q=1, seq_kv=40, kv_len=lens.data_ptr(), lse=lse.data_ptr(),
                mask=mask.data_ptr() if kind else None, stream=torch.cuda.current_stream().cuda_stream)
    h.launch_kv8(**good)
    bad = [dict(kv_len=lens.data_ptr() + 2), dict(lse=lse.data_ptr() + 1), dict(cache=pool.packed(block_table=pool.tab.data_ptr() + 2))]
    if kind == N.MASK_NONE:
        h.launch_kv8(**good, query_starts=starts.data_ptr(), queries=1)
        bad.append(dict(query_starts=starts.data_ptr() + 2, queries=1))
    elif kind == N.MASK_KEEP_U8:
        h.launch_kv8(**{**good, "mask": mask.data_ptr() + 1})
    else:
        bad.append(dict(mask=mask.data_ptr() + 2))
    for b in bad:
        with pytest.raises(N.AidnError) as e:
            h.launch_kv8(**{**good, **b})
        assert e.value.status == N.EINVAL and "aligned" in str(e.value)
    h.poll(torch.cuda.current_stream().cuda_stream)
