"""A paged key / value cache held in 8 bits: the append (rotation, scales, codes) against a restatement that is equal bit for
bit, attention over the cache against the formula in 64 bits.

Tolerances of the attention.  With S = sum |q_d k_d| * scale the largest of a row, u the unit roundoff of the output's type,
A = sum_j p_j |v_j| (what absolute errors of the weights act on):

* products of a query and a code are exact; their sum over D elements in 32 bits is off by at most D 2^-23 S, a query in two 16-bit
  terms (32-bit inputs) by 2^-21 S.  A logit's error e changes every weight by a factor within exp(+-2e), so by 2.1 e at most.
* a weight is rounded to 11 bits (2^-11 of it) for 16-bit results, to two terms (2^-21) for 32-bit ones; its exponential and the
  products with scales add some 2^-21, a sum over keys in 32 bits 2^-20 at most.
* the result is rounded once: u |o|.

So |o - o64| <= u |o| + (w + 2.1 e + 2^-19) A with w = 2^-11 or 2^-21, and the log-sum-exp is off by at most e + 2^-20 (1 + |lse|).
"""
import math

import numpy as np
import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer, KvCacheFp8
from tests._harness import AIDN_DT, TORCH_DT, check_guards, guarded

pytestmark = pytest.mark.gpu


# ---- restatements -----------------------------------------------------------------------------------------------------

def scale_of(m):
    """The smallest power of two from 2^-100 on with m <= 448 times it."""
    e = -100
    if m > 0:
        f, x = math.frexp(m)      # m = f 2^x, f in [1/2, 1); 448 = 7/8 2^9
        e = max(-100, min(119, x - 9 if f <= 0.875 else x - 8))
    return 2.0 ** e


def code_values(x):
    """Nearest E4M3 value in 64 bits, ties to even, +-448 beyond; NaN stays."""
    x = np.asarray(x, np.float64)
    mag = np.minimum(np.abs(x), 1e300)
    step = np.exp2(np.floor(np.log2(np.maximum(mag, 2.0 ** -6))) - 3)
    y = np.minimum(np.rint(mag / step) * step, 448.0)
    return np.where(np.isnan(x), np.nan, np.copysign(y, x))


ALL_CODES = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double().numpy()


class Pool:
    """A pool, its table and (64-bit) contents on the host."""

    def __init__(self, lens, block, heads, dim, seed, spare=2, columns=None, clean=True):
        g = np.random.default_rng(seed)
        self.block, self.heads, self.dim, self.batch = block, heads, dim, len(lens)
        need = [-(-n // block) for n in lens]
        self.columns = columns or max(max(need), 1) + 1
        self.blocks = sum(need) + spare
        order = g.permutation(self.blocks)
        self.table = np.full((self.batch, self.columns), self.blocks + 99, np.int32)   # poison past the end
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.blocks, block, heads, dim)
        self.codes = [g.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]
        if clean:
            for c in self.codes:
                c[(c & 0x7f) == 0x7f] = 0x31
        # magnitudes as of normal values: most of the range below 1/8 of the largest code
        for c in self.codes:
            c[(c & 0x7f) > 0x70] -= 0x28
        self.scales = [np.exp2(g.integers(-9, -5, (self.blocks, heads))).astype(np.float32) for _ in range(2)]

    def cuda(self):
        self.t = [torch.from_numpy(c).cuda() for c in self.codes]
        self.s = [torch.from_numpy(s).cuda() for s in self.scales]
        self.tab = torch.from_numpy(self.table).cuda()
        self.cache = KvCacheFp8(*(GpuBuffer(x) for x in self.t + self.s), self.block, self.heads, self.dim)
        return self

    def rows(self, which, b, n):
        """[n, heads, dim] in 64 bits."""
        at = self.table[b, :-(-n // self.block)]
        v = ALL_CODES[self.codes[which][at]] * self.scales[which][at][:, None, :, None].astype(np.float64)
        return v.reshape(-1, self.heads, self.dim)[:n]

    def packed(self, **kw):
        d = dict(key_pool=self.t[0].data_ptr(), value_pool=self.t[1].data_ptr(), key_scale=self.s[0].data_ptr(),
                 value_scale=self.s[1].data_ptr(), block_table=self.tab.data_ptr(), block_table_stride=self.columns,
                 num_blocks=self.blocks, block_size=self.block, kv_heads=self.heads, head_dim=self.dim)
        return N.kv8_cache(**{**d, **kw})


def attend64(pool, q, lens, counts, heads, *, scale, softcap=0.0, causal=True, keep=None, bias=None):
    """(o, lse, A, S) of q [queries, heads, dim] (64 bits) over the pool."""
    o = np.zeros(q.shape)
    a = np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    top = np.zeros(q.shape[:2])
    r = 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        k, v = pool.rows(0, b, n), pool.rows(1, b, n)
        for h in range(heads):
            kh, vh = k[:, h // (heads // pool.heads)], v[:, h // (heads // pool.heads)]
            qs = q[r:r + c, h]
            with np.errstate(invalid="ignore", over="ignore"):
                s = qs @ kh.T * scale
                mag = np.abs(qs) @ np.abs(kh).T * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if bias is not None:
                s = s + bias[b, h, :c, :n]
            seen = np.ones(s.shape, bool)
            if causal:
                seen = np.arange(n)[None] <= np.arange(c)[:, None] + n - c
            if keep is not None:
                seen = seen & keep[b, h, :c, :n]
            for i in range(c):
                z, w = s[i, seen[i]], vh[seen[i]]
                if len(z):
                    m = z.max()
                    p = np.exp(z - m)
                    l = p.sum()
                    o[r + i, h] = p @ w / l
                    a[r + i, h] = p @ np.abs(w) / l
                    lse[r + i, h] = m + np.log(l)
                    top[r + i, h] = np.nanmax(mag[i, seen[i]])
        r += c
    return o, lse, a, top


def bounds(o, lse, a, top, dtype, out, dim):
    u = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out]
    e = (dim * 2.0 ** -23 + (2.0 ** -21 if dtype == "f32" else 0)) * top
    w = 2.0 ** -21 if out == "f32" else 2.0 ** -11
    tiny = 2.0 ** -24 if out == "f16" else 1e-37   # half the least subnormal of the output
    return u * np.abs(o) + (w + 2.1 * e[..., None] + 2.0 ** -19) * a + tiny, e + 2.0 ** -20 * (1 + np.abs(lse))


def attend(pool, q, lens, counts, heads, *, dtype, out=None, scale=None, softcap=0.0, causal=True, stats=True, path=N.PATH_AUTO,
           uniform=None, workspace=True, max_q=None, max_kv=None, poll=True, q_stride=None, o_stride=None, out_t=None,
           head_begin=0, head_count=0, bottom_right=True, causal_offset=0, packed=None, stream=None, mask=None, mask_kind=N.MASK_NONE,
           mask_stride=(0, 0, 0, 0), handle=None):
    """Runs the kernel; guard words around all that it writes.  Returns (out, lse)."""
    out = out or dtype
    total = sum(counts)
    uniform = (min(counts) == max(counts)) if uniform is None else uniform
    max_q, max_kv = max_q or max(max(counts), 1), max_kv or max(max(lens), 1)
    h = handle or N.Handle(device=0, qkv_dtype=AIDN_DT[dtype], out_dtype=AIDN_DT[out], head_dim=pool.dim, num_q_heads=heads,
                           num_kv_heads=pool.heads, causal=causal, causal_bottom_right=bottom_right, causal_offset=causal_offset,
                           emit_lse=stats, softcap=softcap, path=path, head_begin=head_begin, head_count=head_count, mask_kind=mask_kind)
    guards = []
    if out_t is None:
        flat, out_t = guarded((max(total, 1), heads, pool.dim), TORCH_DT[out], "cuda")
        guards.append((flat, "output"))
    lse = None
    if stats:
        flat, lse = guarded((max(total, 1), heads), torch.float32, "cuda")
        guards.append((flat, "log-sum-exp"))
    need = h.kv8_workspace_bytes(pool.batch, max_q, max_kv) if workspace else 0
    flat, ws = guarded((max(need // 4, 4),), torch.float32, "cuda", fill=float("nan"))
    guards.append((flat, "workspace"))
    starts = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    ends = torch.tensor(lens, dtype=torch.int32, device="cuda")
    row = (max_q * heads * pool.dim, pool.dim, heads * pool.dim) if uniform else None
    st = stream or torch.cuda.current_stream().cuda_stream
    h.launch_kv8(q=q.data_ptr(), out=out_t.data_ptr(), cache=packed or pool.packed(), batch=pool.batch, seq_q=max_q, seq_kv=max_kv,
                 stream=st, query_starts=None if uniform else starts.data_ptr(), queries=total, lse=lse.data_ptr() if stats else None,
                 kv_len=ends.data_ptr(), q_stride=q_stride or row, o_stride=o_stride or row, scale=scale or 0.0,
                 workspace=ws.data_ptr() if need else None, workspace_bytes=need, mask=mask.data_ptr() if mask is not None else None,
                 mask_stride=mask_stride)
    if poll:
        h.poll(st)
        for flat, what in guards:
            check_guards(flat, what)
    return out_t, lse


def check(pool, q, lens, counts, heads, *, dtype, out=None, softcap=0.0, causal=True, got=None, **kw):
    out = out or dtype
    scale = kw.get("scale") or 1 / math.sqrt(pool.dim)
    o, lse, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, heads, scale=scale, softcap=softcap, causal=causal)
    bo, bl = bounds(o, lse, a, top, dtype, out, pool.dim)
    go, gl = got or attend(pool, q, lens, counts, heads, dtype=dtype, out=out, softcap=softcap, causal=causal, **kw)
    go, gl = go.double().cpu().numpy()[:len(o)], gl.double().cpu().numpy()[:len(o)]
    off = np.abs(go - o) - bo
    assert np.isfinite(go).all()
    assert off.max(initial=-1) <= 0, f"output off by {np.abs(go - o).max():.3e}, {off.max():.3e} over its bound"
    assert np.array_equal(np.isneginf(gl), np.isneginf(lse))
    seen = ~np.isneginf(lse)
    off = np.abs(gl[seen] - lse[seen]) - bl[seen]
    assert off.max(initial=-1) <= 0, f"log-sum-exp {off.max():.3e} over its bound"
    return go, gl


def queries(n, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((n, heads, dim), generator=g).to(TORCH_DT[dtype]).cuda()


# ---- attention ---------------------------------------------------------------------------------------------------------

SHAPES = [
    # lens, counts, heads, kv_heads, dim, block
    ([1], [1], 1, 1, 64, 16),
    ([17], [1], 8, 8, 128, 16),
    ([16, 15, 33, 128, 129], [1] * 5, 8, 2, 128, 16),
    ([700, 3, 1500], [1] * 3, 12, 4, 64, 32),
    ([300, 257], [1] * 2, 32, 2, 128, 64),
    ([511], [1], 20, 1, 128, 128),
    ([77, 1030], [1] * 2, 6, 2, 128, 8),
    ([77, 1030], [1] * 2, 6, 2, 64, 24),
    ([100, 200], [1] * 2, 4, 2, 96, 16),
    ([100, 333], [1] * 2, 4, 1, 256, 16),
    ([50, 60], [1] * 2, 3, 3, 40, 5),
    ([65, 300, 1000], [3] * 3, 8, 2, 128, 16),
    ([8, 300, 1000], [8, 1, 5], 8, 2, 64, 16),
    ([40, 300], [7, 6], 14, 2, 128, 16),
    ([260, 131], [70, 131], 8, 4, 64, 32),
    ([700], [257], 8, 2, 128, 16),
    ([900, 40, 513], [300, 1, 128], 16, 4, 128, 64),
    ([333, 1000], [100, 333], 4, 4, 64, 128),
    ([129, 65], [129, 33], 6, 2, 256, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"n{'_'.join(map(str, s[0]))}q{'_'.join(map(str, s[1]))}h{s[2]}kv{s[3]}d{s[4]}b{s[5]}")
@pytest.mark.parametrize("path", [N.PATH_AUTO, N.PATH_GENERIC], ids=["auto", "generic"])
def test_attention(shape, dtype, path):
    lens, counts, heads, kv, dim, block = shape
    pool = Pool(lens, block, kv, dim, seed=sum(lens) + dim).cuda()
    check(pool, queries(sum(counts), heads, dim, dtype, 5), lens, counts, heads, dtype=dtype, path=path)


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("counts", [[1, 1, 1], [4, 4, 4], [90, 1, 200]])
def test_attention_fp32_results(dtype, out, counts):
    lens = [300, 1, 1200]
    counts = [min(c, n) for c, n in zip(counts, lens)]
    pool = Pool(lens, 16, 2, 128, seed=3).cuda()
    check(pool, queries(sum(counts), 8, 128, dtype, 6), lens, counts, 8, dtype=dtype, out=out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1], [5, 5], [150, 60]])
def test_softcap(dtype, counts):
    lens = [900, 77]
    pool = Pool(lens, 16, 2, 64, seed=4).cuda()
    check(pool, queries(sum(counts), 8, 64, dtype, 7) * 4, lens, counts, 8, dtype=dtype, softcap=5.0)


@pytest.mark.parametrize("counts", [[1, 1], [6, 3], [150, 60]])
def test_not_causal(counts):
    lens = [900, 177]
    pool = Pool(lens, 16, 2, 128, seed=4).cuda()
    check(pool, queries(sum(counts), 8, 128, "f16", 7), lens, counts, 8, dtype="f16", causal=False)


@pytest.mark.parametrize("counts,causal", [([1, 1, 1, 1], True), ([4, 2, 6, 3], True), ([200, 4, 140, 3], True), ([200, 4, 140, 3], False)])
def test_rows_without_keys(counts, causal):
    """No keys at all, and fewer keys than queries: zeros and -inf, for the rows that see none alone."""
    lens = [500, 0, 3, 0]
    pool = Pool(lens, 16, 2, 128, seed=9).cuda()
    check(pool, queries(sum(counts), 8, 128, "bf16", 8), lens, counts, 8, dtype="bf16", causal=causal)


def test_sequences_without_queries():
    lens, counts = [100, 300, 50, 70, 9], [0, 5, 0, 0, 1]
    pool = Pool(lens, 16, 2, 64, seed=10).cuda()
    check(pool, queries(6, 4, 64, "f16", 8), lens, counts, 4, dtype="f16", uniform=False)


@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [130, 200]])
@pytest.mark.parametrize("block", [16, 24, 128])
def test_what_lies_past_the_end(counts, block):
    """NaN codes and NaN scales in rows and blocks past a sequence's keys reach nothing."""
    lens = [457, 205]
    pool = Pool(lens, block, 2, 128, seed=11)
    q = queries(sum(counts), 8, 128, "bf16", 9)
    clean = attend(pool.cuda(), q, lens, counts, 8, dtype="bf16")
    used = {int(pool.table[b, j]) for b, n in enumerate(lens) for j in range(-(-n // block))}
    for c, s in zip(pool.codes, pool.scales):
        for blk in set(range(pool.blocks)) - used:
            c[blk], s[blk] = 0x7f, np.nan
        for b, n in enumerate(lens):
            if n % block:
                c[pool.table[b, n // block], n % block:] = 0xff
    dirty = attend(pool.cuda(), q, lens, counts, 8, dtype="bf16")
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("counts", [[4, 4], [150, 70]])
@pytest.mark.parametrize("which", [0, 1])
def test_nan_in_keys_that_some_queries_do_not_see(counts, which):
    """A NaN key or value makes the rows that see it NaN and leaves the others as they are."""
    lens = [300, 100]
    pool = Pool(lens, 16, 2, 64, seed=12).cuda()
    q = queries(sum(counts), 4, 64, "f16", 9)
    clean, _ = attend(pool, q, lens, counts, 4, dtype="f16")
    first = counts[0] // 2     # of sequence 0: the first query that sees the key
    key = lens[0] - counts[0] + first
    pool.codes[which][pool.table[0, key // 16], key % 16, 1, 7] = 0x7f
    dirty, _ = attend(pool.cuda(), q, lens, counts, 4, dtype="f16")
    hit = torch.zeros(clean.shape[:2], dtype=torch.bool)
    hit[first:counts[0], 2:4] = True
    assert dirty.isnan().any(-1).cpu().equal(hit)
    assert torch.equal(clean[~hit.cuda()], dirty[~hit.cuda()])


@pytest.mark.parametrize("counts", [[1, 1], [5, 5], [130, 130]])
def test_scales_far_apart(counts):
    """Blocks whose scales differ by up to 2^24, and any positive scale, not only powers of two."""
    lens = [400, 210]
    pool = Pool(lens, 16, 2, 128, seed=13)
    g = np.random.default_rng(1)
    pool.scales[1] = (np.exp2(g.integers(-20, 5, pool.scales[1].shape)) * g.uniform(1, 2, pool.scales[1].shape)).astype(np.float32)
    pool.scales[0] = (pool.scales[0] * g.uniform(0.1, 2, pool.scales[0].shape)).astype(np.float32)
    for dtype in ("f16", "f32"):
        check(pool.cuda(), queries(sum(counts), 8, 128, dtype, 10), lens, counts, 8, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("exponent", [-60, 40])
def test_queries_of_extreme_size(dtype, exponent):
    """Queries outside what 16 bits hold, the logits brought back by the scale."""
    lens, counts = [300, 90], [2, 2]
    pool = Pool(lens, 16, 2, 128, seed=14).cuda()
    q = (queries(4, 4, 128, "bf16", 11).float() * 2.0 ** exponent).to(TORCH_DT[dtype])
    check(pool, q, lens, counts, 4, dtype=dtype, scale=2.0 ** -exponent / 11)


def test_zero_queries_and_large_logits():
    lens, counts = [300, 90], [2, 130 - 100]
    pool = Pool(lens, 16, 2, 128, seed=15).cuda()
    q = queries(sum(counts), 4, 128, "f16", 12) * 30
    q[0] = 0
    check(pool, q, lens, counts, 4, dtype="f16")


@pytest.mark.parametrize("counts", [[1, 1], [4, 4], [140, 140]])
def test_strided_tensors(counts):
    """Queries inside a wider packed tensor, results into another; pools with the heads outside the tokens."""
    lens = [300, 290]
    pool = Pool(lens, 16, 2, 64, seed=16).cuda()
    q = queries(sum(counts), 8, 64, "bf16", 13)
    plain = attend(pool, q, lens, counts, 8, dtype="bf16")
    n = counts[0]
    wide = torch.full((sum(counts), 12, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, :8, :64] = q
    into = torch.full((sum(counts), 9, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    moved = [t.transpose(1, 2).contiguous() for t in pool.t]   # [blocks, heads, tokens, dim]
    packed = pool.packed(key_pool=moved[0].data_ptr(), value_pool=moved[1].data_ptr(), pool_stride=(2 * 16 * 64, 64, 16 * 64))
    attend(pool, wide, lens, counts, 8, dtype="bf16", q_stride=(n * 12 * 72, 72, 12 * 72), o_stride=(n * 9 * 64, 64, 9 * 64),
           out_t=into, packed=packed)
    assert torch.equal(into[:, :8], plain[0]) and bool((into[:, 8] == 5.0).all())


def test_unaligned_queries_and_pools():
    """Rows that start anywhere their elements may: queries two bytes off, pools four."""
    lens, counts = [300, 90], [3, 3]
    pool = Pool(lens, 16, 2, 64, seed=17).cuda()
    q = queries(6, 4, 64, "f16", 14)
    off = torch.empty(q.numel() + 1, dtype=torch.float16, device="cuda")
    off[1:] = q.flatten()
    pools = []
    for t in pool.t:
        pools.append(torch.zeros(t.numel() + 4, dtype=torch.uint8, device="cuda"))
        pools[-1][4:] = t.flatten()
    packed = pool.packed(key_pool=pools[0].data_ptr() + 4, value_pool=pools[1].data_ptr() + 4)
    got = attend(pool, off[1:], lens, counts, 4, dtype="f16", packed=packed)
    check(pool, q, lens, counts, 4, dtype="f16", got=got)


def test_offsets_past_32_bits():
    """Blocks beyond the first 4 GiB of the pools."""
    lens, counts, kv, dim, block = [100, 300], [1, 40], 2, 128, 16
    per = block * kv * dim
    base = (1 << 32) // per + 5
    pool = Pool(lens, block, kv, dim, seed=18).cuda()
    big = [torch.empty((base + pool.blocks) * per, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full(((base + pool.blocks), kv), float("nan"), device="cuda") for _ in range(2)]
    for i in range(2):
        big[i][base * per:] = pool.t[i].flatten()
        scales[i][base:] = pool.s[i]
    tab = pool.tab + base
    packed = pool.packed(key_pool=big[0].data_ptr(), value_pool=big[1].data_ptr(), key_scale=scales[0].data_ptr(),
                         value_scale=scales[1].data_ptr(), block_table=tab.data_ptr(), num_blocks=base + pool.blocks)
    q = queries(sum(counts), 4, dim, "bf16", 15)
    got = attend(pool, q, lens, counts, 4, dtype="bf16", packed=packed)
    check(pool, q, lens, counts, 4, dtype="bf16", got=got)


@pytest.mark.parametrize("counts", [[1, 1], [150, 150]])
def test_table_entries_outside_the_pool(counts):
    """A bad entry is reported by poll, never followed; its keys count for nothing."""
    lens = [320, 200]
    pool = Pool(lens, 16, 2, 64, seed=19)
    pool.table[0, 7] = pool.blocks + 3
    pool.table[1, 2] = -1
    pool.cuda()
    h = N.Handle(device=0, qkv_dtype=N.F16, out_dtype=N.F16, head_dim=64, num_q_heads=4, num_kv_heads=2, causal=True, emit_lse=True)
    out, _ = attend(pool, queries(sum(counts), 4, 64, "f16", 16), lens, counts, 4, dtype="f16", handle=h, poll=False)
    with pytest.raises(N.AidnError) as e:
        h.poll(torch.cuda.current_stream().cuda_stream)
    assert e.value.status == N.EINVAL and bool(out.isfinite().all())


@pytest.mark.parametrize("counts", [[1] * 4, [3] * 4, [130, 1, 64, 200]])
def test_without_workspace_and_again(counts):
    """No workspace: keys are not cut, the result is within the same bounds; the same call twice gives the same bits, and a call with other
    lengths between leaves nothing behind."""
    lens = [2000, 777, 64, 1500]
    pool = Pool(lens, 16, 2, 128, seed=20).cuda()
    q = queries(sum(counts), 8, 128, "bf16", 17)
    check(pool, q, lens, counts, 8, dtype="bf16", workspace=False)
    h = N.Handle(device=0, qkv_dtype=N.BF16, out_dtype=N.BF16, head_dim=128, num_q_heads=8, num_kv_heads=2, causal=True, emit_lse=True)
    a = attend(pool, q, lens, counts, 8, dtype="bf16", handle=h)
    attend(pool, q, [min(n, c + 9) for n, c in zip(lens, counts)], counts, 8, dtype="bf16", handle=h)
    b = attend(pool, q, lens, counts, 8, dtype="bf16", handle=h)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(pool, q, lens, counts, 8, dtype="bf16", got=b)


@pytest.mark.parametrize("counts", [[1, 1], [140, 33]])
def test_head_shards(counts):
    lens = [500, 321]
    pool = Pool(lens, 16, 4, 64, seed=21).cuda()
    q = queries(sum(counts), 8, 64, "f16", 18)
    whole = attend(pool, q, lens, counts, 8, dtype="f16", workspace=False)
    flat, part = guarded((sum(counts), 8, 64), torch.float16, "cuda", fill=0.0)
    for begin, n in ((0, 2), (2, 4), (6, 2)):
        attend(pool, q, lens, counts, 8, dtype="f16", workspace=False, head_begin=begin, head_count=n, out_t=part, stats=False)
    check_guards(flat, "output")
    assert torch.equal(part, whole[0])


@pytest.mark.parametrize("counts", [1, 5, 60])
@pytest.mark.parametrize("offset", [0, 37])
def test_top_left_causal(counts, offset):
    """causal_bottom_right = 0: query i sees keys up to i + causal_offset, whatever the lengths."""
    lens = [150, 90]
    pool = Pool(lens, 16, 2, 64, seed=22).cuda()
    q = queries(2 * counts, 4, 64, "f16", 19)
    got, _ = attend(pool, q, lens, [counts] * 2, 4, dtype="f16", bottom_right=False, causal_offset=offset)
    for b in range(2):
        for i in range(0, counts, 7):
            n = min(lens[b], i + offset + 1)
            one, _ = attend(Pool(lens, 16, 2, 64, seed=22).cuda(), q[b * counts + i].repeat(2, 1, 1), [n, n] if b == 0 else [1, n], [1, 1], 4, dtype="f16", path=N.PATH_GENERIC)
            assert (one[b].float() - got[b * counts + i].float()).abs().max() <= 2.0 ** -9 * got[b * counts + i].float().abs().max()


@pytest.mark.parametrize("kind", [N.MASK_KEEP_U8, N.MASK_KEEP_F32, N.MASK_ADD_F32])
def test_masks(kind):
    """Masks over (b, h, i, j), one row of which keeps nothing, one holds the lowest value, one NaN and inf in masked places."""
    lens, counts, heads = [90, 70], [4, 4], 4
    pool = Pool(lens, 16, 2, 64, seed=23).cuda()
    q = queries(8, heads, 64, "f32", 20)
    g = np.random.default_rng(3)
    keep = g.random((2, heads, 4, 90)) < 0.6
    keep[0, 1, 2] = False
    keep[..., 0] |= np.arange(4)[None, None] != 2
    bias = None
    if kind == N.MASK_ADD_F32:
        bias = np.where(keep, g.standard_normal(keep.shape), -np.inf).astype(np.float32)
        bias[1, 0, 0] = np.where(keep[1, 0, 0], bias[1, 0, 0], np.finfo(np.float32).min)
        mask = torch.from_numpy(bias).cuda()
    else:
        mask = torch.from_numpy(keep).cuda().to(torch.uint8 if kind == N.MASK_KEEP_U8 else torch.float32).contiguous()
    got, lse = attend(pool, q, lens, counts, heads, dtype="f32", mask=mask, mask_kind=kind, mask_stride=mask.stride())
    o, ref, a, top = attend64(pool, q.double().cpu().numpy(), lens, counts, heads, scale=1 / 8, keep=keep,
                              bias=None if bias is None else np.where(keep, bias, 0))
    bo, bl = bounds(o, ref, a, top, "f32", "f32", 64)
    assert (np.abs(got.double().cpu().numpy() - o) <= bo).all()
    lse = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(lse), np.isneginf(ref))
    assert (np.abs(lse - ref)[~np.isneginf(ref)] <= bl[~np.isneginf(ref)]).all()


def test_graph_and_streams():
    """Append and attention captured together on a side stream, replayed twice over new inputs."""
    be = CudaBackend(0)
    cache = be.AllocateKvCacheFp8(40, 16, 2, 128)
    table = GpuBuffer(torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 20).cuda())
    start, ends = GpuBuffer(torch.tensor([0, 0], dtype=torch.int32).cuda()), GpuBuffer(torch.tensor([250, 250], dtype=torch.int32).cuda())
    ctx = GpuBuffer(torch.randn((500, 8, 128), generator=torch.Generator().manual_seed(2)).bfloat16().cuda())
    be.PagedKvAppendFp8(ctx, GpuBuffer(torch.empty(500, 4, 128).bfloat16().cuda()), cache, table, start, 2, 500, 4, 20)
    step = torch.randn((3, 2, 8, 128), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    at = GpuBuffer(torch.tensor([250, 250], dtype=torch.int32).cuda())
    ends.tensor += 1
    x, q, out = (GpuBuffer(torch.zeros((2, n, 128)).bfloat16().cuda()) for n in (8, 4, 4))

    def run():
        be.PagedKvAppendFp8(x, q, cache, table, at, 2, 2, 4, 20)
        be.PagedAttentionFp8(q, cache, table, ends, out, 2, 4, 1, 320, 20, 0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.tensor.copy_(step[0])
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for i in (1, 2):
        x.tensor.copy_(step[i])
        graph.replay()
        torch.cuda.synchronize()
        got = out.tensor.clone()
        out.tensor.zero_()
        run()
        torch.cuda.synchronize()
        assert torch.equal(got, out.tensor) and bool(got.isfinite().all())
        q64 = step[i, :, :4].double()
        for b in range(2):
            k = torch.cat([ctx.tensor[b * 250:(b + 1) * 250], step[i, b:b + 1]]).double()
            z = torch.einsum("hd,jhd->hj", q64[b], k[:, 4:6].repeat_interleave(2, 1)) * 0.1
            o = torch.einsum("hj,jhd->hd", z.softmax(-1), k[:, 6:].repeat_interleave(2, 1))
            assert (o - got[b].double()).abs().max() < 0.25   # three-bit codes against none: rounding of up to 2^-4 of a value


def test_refusals():
    be = CudaBackend(0)
    pool = Pool([40], 16, 2, 64, seed=1).cuda()
    q = GpuBuffer(queries(1, 4, 64, "bf16", 1))
    lens, table, out = GpuBuffer(torch.tensor([40], dtype=torch.int32).cuda()), GpuBuffer(pool.tab), GpuBuffer(torch.empty(4 * 64).bfloat16().cuda())

    def call(**kw):
        a = dict(q=q, cache=pool.cache, blockTables=table, seqLens=lens, output=out, batch=1, heads=4, maxQueries=1, maxSeqLen=40,
                 blocksPerSeq=pool.columns, scale=0.1)
        be.PagedAttentionFp8(**{**a, **kw})

    call()
    for bad in (dict(heads=3), dict(heads=0), dict(batch=0), dict(maxQueries=0), dict(maxSeqLen=0), dict(blocksPerSeq=0), dict(maxQueries=2),
                dict(batch=2), dict(seqLens=GpuBuffer(lens.tensor.float())), dict(output=GpuBuffer(out.tensor[:100].clone())),
                dict(softmaxStats=GpuBuffer(torch.empty(3).cuda())), dict(queryStarts=GpuBuffer(torch.zeros(1, dtype=torch.int32).cuda())),
                dict(blockTables=GpuBuffer(table.tensor[:, :1].contiguous()))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):
        KvCacheFp8(pool.cache.keys, pool.cache.values, pool.cache.keyScales, pool.cache.valueScales, 16, 2, 60)
    with pytest.raises(ValueError):
        KvCacheFp8(pool.cache.keys, pool.cache.values, GpuBuffer(pool.s[0][:1].clone()), pool.cache.valueScales, 16, 2, 64)
    h = N.Handle(device=0, qkv_dtype=N.BF16, out_dtype=N.BF16, head_dim=64, num_q_heads=4, num_kv_heads=2, causal=True)
    good = dict(q=q.Handle, out=out.Handle, cache=pool.packed(), batch=1, seq_q=1, seq_kv=40, kv_len=lens.Handle,
                stream=torch.cuda.current_stream().cuda_stream)
    h.launch_kv8(**good)
    for bad, status in ((dict(q=0), N.EINVAL), (dict(batch=0), N.EINVAL), (dict(seq_kv=0), N.EINVAL), (dict(scale=-1.0), N.EINVAL),
                        (dict(cache=pool.packed(kv_heads=4)), N.EINVAL), (dict(cache=pool.packed(head_dim=128)), N.EINVAL),
                        (dict(cache=pool.packed(block_size=0)), N.EINVAL), (dict(cache=pool.packed(key_scale=0)), N.EINVAL),
                        (dict(cache=pool.packed(block_table_stride=0)), N.EINVAL), (dict(cache=pool.packed(pool_stride=(2048, 130, 64))), N.EINVAL),
                        (dict(query_starts=lens.Handle, queries=0), N.EINVAL), (dict(q_stride=(64, -64, 64)), N.EINVAL),
                        (dict(q=q.Handle + 1), N.EINVAL)):
        with pytest.raises(N.AidnError) as e:
            h.launch_kv8(**{**good, **bad})
        assert e.value.status == status, bad


# ---- append -------------------------------------------------------------------------------------------------------------

def turn(x, cos, sin, interleaved):
    """fp32, every operation rounded on its own.  x [n, heads, dim]."""
    c, s = cos[:, None], sin[:, None]
    y = x.copy()
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    with np.errstate(invalid="ignore", over="ignore"):
        u, w = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0::2], y[..., 1::2] = u, w
    else:
        y[..., :half], y[..., half:] = u, w
    return y


def append_ref(pool, which, rows, b, start):
    """Puts rows [n, heads, dim] (fp32) of sequence b into the host's pool."""
    size = pool.block
    for j in range(start // size, (start + len(rows) - 1) // size + 1):
        at = pool.table[b, j]
        low, high = max(start, j * size), min(start + len(rows), (j + 1) * size)
        part, had = rows[low - start:high - start], low - j * size
        for h in range(pool.heads):
            m = np.abs(part[:, h])
            s = scale_of(float(m[np.isfinite(m)].max(initial=0)))
            old = float(pool.scales[which][at, h])
            if had and old >= s:
                s = old
            elif had:
                pool.codes[which][at, :had, h] = encode(ALL_CODES[pool.codes[which][at, :had, h]] * (old / s))
            pool.scales[which][at, h] = s
            pool.codes[which][at, had:high - j * size, h] = encode(part[:, h].astype(np.float64) / s)


FINITE = [i for i in range(256) if i & 0x7f != 0x7f]


def encode(x):
    v = code_values(x)
    order = sorted(FINITE[:127], key=lambda i: ALL_CODES[i])
    mag = np.abs(np.where(np.isnan(v), 0, v))
    c = np.asarray(order, np.uint8)[np.searchsorted(ALL_CODES[order], mag)]
    return np.where(np.isnan(v), 0x7f, c | (np.signbit(v).astype(np.uint8) << 7)).astype(np.uint8)


def same_codes(a, b):
    """Equal bytes, or NaN both."""
    nan = (a & 0x7f) == 0x7f
    return np.array_equal(nan, (b & 0x7f) == 0x7f) and np.array_equal(a[~nan], b[~nan])


APPENDS = [
    # starts, counts, heads, kv_heads, dim, block
    ([0], [1], 4, 2, 128, 16),
    ([5], [1], 1, 1, 64, 16),
    ([0, 15, 16, 100], [1] * 4, 32, 8, 128, 16),
    ([0, 3, 40], [33, 16, 13], 4, 2, 64, 16),
    ([7, 0], [100, 100], 8, 2, 128, 32),
    ([50, 0, 1], [3, 300, 129], 6, 3, 128, 128),
    ([2, 9], [50, 20], 4, 2, 256, 64),
    ([2, 9], [50, 20], 5, 1, 96, 24),
    ([1, 0], [17, 4], 3, 3, 40, 5),
    ([0, 600], [520, 300], 2, 2, 64, 512),
    ([3, 0, 8, 0], [0, 5, 0, 20], 2, 1, 128, 8),
    ([11] * 70, [2] * 70, 2, 2, 64, 16),
]


@pytest.mark.parametrize("shape", APPENDS, ids=lambda s: f"s{'_'.join(map(str, s[0][:4]))}n{'_'.join(map(str, s[1][:4]))}h{s[2]}kv{s[3]}d{s[4]}b{s[5]}")
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rope", ["none", "interleaved", "halves"])
def test_append(shape, dtype, rope):
    starts, counts, heads, kv, dim, block = shape
    ends = [a + n for a, n in zip(starts, counts)]
    pool = Pool(ends, block, kv, dim, seed=sum(ends) + dim).cuda()
    g = torch.Generator().manual_seed(7)
    tokens = sum(counts)
    x = (torch.randn((tokens, heads + 2 * kv, dim), generator=g) * torch.exp2(torch.randint(-6, 4, (tokens, 1, 1), generator=g))).to(TORCH_DT[dtype])
    cos, sin = torch.rand((2, max(ends) + 1, dim // 2), generator=g) * 2 - 1
    be = CudaBackend(0)
    flat, q = guarded((tokens, heads, dim), TORCH_DT[dtype], "cuda")
    cu = GpuBuffer(torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda())
    be.PagedKvAppendFp8(GpuBuffer(x.cuda()), GpuBuffer(q), pool.cache, GpuBuffer(pool.tab), GpuBuffer(torch.tensor(starts, dtype=torch.int32).cuda()),
                        len(starts), tokens, heads, pool.columns, cos=None if rope == "none" else GpuBuffer(cos.cuda()),
                        sin=None if rope == "none" else GpuBuffer(sin.cuda()), interleaved=rope == "interleaved",
                        tokenStarts=None if min(counts) == max(counts) else cu)
    torch.cuda.synchronize()
    check_guards(flat, "queries")
    r = 0
    for b, (a, n) in enumerate(zip(starts, counts)):
        if n == 0:
            continue
        f = x[r:r + n].float().numpy()
        qk = f[:, :heads + kv]
        if rope != "none":
            qk = turn(qk, cos[a:a + n].numpy(), sin[a:a + n].numpy(), rope == "interleaved")
        assert torch.equal(q[r:r + n].cpu(), torch.from_numpy(qk[:, :heads].copy()).to(TORCH_DT[dtype]))
        append_ref(pool, 0, qk[:, heads:], b, a)
        append_ref(pool, 1, f[:, heads + kv:], b, a)
        r += n
    for i in range(2):
        assert np.array_equal(pool.s[i].cpu().numpy(), pool.scales[i])
        assert same_codes(pool.t[i].cpu().numpy(), pool.codes[i])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_of_special_values(dtype):
    """Zeros, subnormals, NaN, infinities, the largest floats, and magnitudes at the edge of a scale."""
    kinds = [0.0, 1e-40, 2.0 ** -100, 448.0, 449.0, 1.75 * 2.0 ** 30, 1.7500002 * 2.0 ** 30, 3.3e38, 7.0]
    starts, n, dim = [0, 4] * len(kinds), 3, 64
    pool = Pool([s + n for s in starts], 8, 1, dim, seed=2).cuda()
    x = torch.randn((len(starts) * n, 2, dim), generator=torch.Generator().manual_seed(1))
    for b in range(len(starts)):
        part = x[b * n:(b + 1) * n]
        part *= kinds[b // 2] / part.abs().amax()
        part[0, :, 3] = kinds[b // 2]
        part[1, :, 5], part[1, :, 6], part[2, :, 7] = float("nan"), float("inf"), -float("inf")
    x = x.to(TORCH_DT[dtype])
    CudaBackend(0).PagedKvAppendFp8(GpuBuffer(x.cuda()), None, pool.cache, GpuBuffer(pool.tab), GpuBuffer(torch.tensor(starts, dtype=torch.int32).cuda()),
                                    len(starts), len(x), 0, pool.columns)
    torch.cuda.synchronize()
    for b, a in enumerate(starts):
        for i in range(2):
            append_ref(pool, i, x[b * n:(b + 1) * n, i:i + 1].float().numpy(), b, a)
    for i in range(2):
        assert np.array_equal(pool.s[i].cpu().numpy(), pool.scales[i])
        assert same_codes(pool.t[i].cpu().numpy(), pool.codes[i])


def test_append_keeps_to_its_rows():
    """Bad table entries, sequences past their table and negative starts are skipped; in-place rotation of a packed tensor that is not
    16-byte aligned; rotation positions of their own."""
    starts, counts, heads, kv, dim, block = [3, -1, 0, 30], [4] * 4, 2, 1, 64, 16
    pool = Pool([48] * 4, block, kv, dim, seed=3, columns=3)
    pool.table[2, 0] = pool.blocks
    pool.cuda()
    before = [t.clone() for t in pool.t]
    g = torch.Generator().manual_seed(4)
    x = torch.randn((16, heads + 2 * kv, dim), generator=g).half()
    cos, sin = torch.rand((2, 9, dim // 2), generator=g)
    places = torch.tensor([0, 3, 8, 9, -1] + list(range(11)), dtype=torch.int32)   # 9 and more, and -1, are outside
    off = torch.zeros(x.numel() + 3, dtype=torch.half, device="cuda")
    off[3:] = x.cuda().flatten()
    at, size, row = off.data_ptr() + 6, 2 * dim, (4 * dim, dim)
    c, s, pl, st = cos.cuda(), sin.cuda(), places.cuda(), torch.tensor([3, -1, 0, 46], dtype=torch.int32).cuda()
    N.kv8_append(pool.packed(), query=at, query_out=at, key=at + heads * size, value=at + (heads + 1) * size, heads=heads, start=st.data_ptr(),
                 tokens=16, batch=4, dtype=N.F16, cosine=c.data_ptr(), sine=s.data_ptr(), rope=N.ROPE_HALVES, max_position=9,
                 positions=pl.data_ptr(), query_stride=row, key_stride=row, value_stride=row, query_out_stride=row,
                 stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    f = x.float().numpy()
    inside = [0 <= p < 9 for p in places.tolist()]
    t = turn(f[:, :3], cos.numpy()[np.clip(places.numpy(), 0, 8)], sin.numpy()[np.clip(places.numpy(), 0, 8)], False)
    t = np.where(np.array(inside)[:, None, None], t, f[:, :3])
    got = off[3:].view(16, 4, dim).cpu()
    assert torch.equal(got[:, :2], torch.from_numpy(t[:, :2].copy()).half()) and torch.equal(got[:, 2:], x[:, 2:])
    append_ref(pool, 0, t[:4, 2:], 0, 3)
    append_ref(pool, 1, f[:4, 3:], 0, 3)
    append_ref(pool, 0, t[12:14, 2:], 3, 46)     # positions 48 and 49 are past the table
    append_ref(pool, 1, f[12:14, 3:], 3, 46)
    for i in range(2):
        assert same_codes(pool.t[i].cpu().numpy(), pool.codes[i])
        assert not torch.equal(pool.t[i], before[i])


def test_append_token_by_token_equals_itself_in_blocks():
    """One call a token against one call for all: the same scales; codes off by what the moves round alone."""
    n, kv, dim, block = 61, 2, 128, 16
    x = torch.randn((n, 2 * kv, dim), generator=torch.Generator().manual_seed(5)) * torch.exp2(torch.arange(n)[:, None, None] % 7 - 3.0)
    pools = [Pool([n], block, kv, dim, seed=6).cuda() for _ in range(2)]
    be = CudaBackend(0)
    be.PagedKvAppendFp8(GpuBuffer(x.cuda()), None, pools[0].cache, GpuBuffer(pools[0].tab), GpuBuffer(torch.zeros(1, dtype=torch.int32).cuda()), 1, n, 0, pools[0].columns)
    for i in range(n):
        be.PagedKvAppendFp8(GpuBuffer(x[i:i + 1].cuda()), None, pools[1].cache, GpuBuffer(pools[1].tab), GpuBuffer(torch.tensor([i], dtype=torch.int32).cuda()), 1, 1, 0,
                            pools[1].columns)
    torch.cuda.synchronize()
    for p in pools:
        p.codes, p.scales = [t.cpu().numpy() for t in p.t], [s.cpu().numpy() for s in p.s]
    for i in range(2):
        used = pools[0].table[0, :4]
        assert np.array_equal(pools[0].scales[i][used], pools[1].scales[i][used])
        a, b = pools[0].rows(i, 0, n), pools[1].rows(i, 0, n)
        step = np.repeat(pools[0].scales[i][used], block, 0)[:n, :, None] * 2.0 ** -9   # the least step of a code
        assert (np.abs(a - b) <= step).all()


def test_append_refusals():
    pool = Pool([40], 16, 2, 64, seed=1).cuda()
    x = torch.randn(3, 6, 64).half().cuda()
    st = torch.zeros(1, dtype=torch.int32).cuda()
    good = dict(key=x.data_ptr(), value=x.data_ptr(), start=st.data_ptr(), tokens=3, batch=1, dtype=N.F16,
                stream=torch.cuda.current_stream().cuda_stream)
    N.kv8_append(pool.packed(), **good)
    for bad in (dict(key=0), dict(value=0), dict(start=0), dict(tokens=-1), dict(batch=0), dict(batch=2), dict(dtype=7), dict(rope=3),
                dict(rope=1), dict(query=x.data_ptr()), dict(query=x.data_ptr(), query_out=x.data_ptr()), dict(key=x.data_ptr() + 1),
                dict(key_stride=(-64, 64))):
        with pytest.raises(N.AidnError) as e:
            N.kv8_append(pool.packed(), **{**good, **bad})
        assert e.value.status == N.EINVAL, bad
    for bad, status in ((dict(block_size=0), N.EINVAL), (dict(head_dim=60), N.EUNSUPPORTED), (dict(head_dim=264), N.EINVAL), (dict(block_table=0), N.EINVAL),
                        (dict(block_table_stride=0), N.EINVAL), (dict(num_blocks=-1), N.EINVAL)):
        with pytest.raises(N.AidnError) as e:
            N.kv8_append(pool.packed(**bad), **good)
        assert e.value.status == status, bad
    be = CudaBackend(0)
    for bad in (dict(heads=5), dict(tokens=4), dict(batch=2), dict(queries=None), dict(cos=GpuBuffer(torch.ones(64).cuda())), dict(blocksPerSeq=0)):
        a = dict(qkv=GpuBuffer(x), queries=GpuBuffer(torch.empty(3, 2, 64).half().cuda()), cache=pool.cache, blockTables=GpuBuffer(pool.tab),
                 startLens=GpuBuffer(st), batch=1, tokens=3, heads=2, blocksPerSeq=pool.columns)
        with pytest.raises(ValueError):
            be.PagedKvAppendFp8(**{**a, **bad})
