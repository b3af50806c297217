"""Linear attention with a decay for each head (prompts, gradients, single tokens) against the recurrence in 64 bits.

Bounds.  u is the unit roundoff of the type (0 where it is fp32: the products are not rounded there), |x|-quantities are the same recurrence over absolute
values: A_t = scale * |q_t| S|_t with S|_t = exp(g) S|_(t-1) + |k_t| |v_t|^T.  Every rounding of a product, weight or state acts on a
term of A:

* 16-bit types: weighted products q . k, and states where they meet queries, are rounded to the type: u A between them (a term goes through one of the
  two).  The type's smallest numbers are no limit: both are scaled to their own size first.
* a weighted key is held in two terms of the type: 4 u^2 of S| for states.
* fp32 sums: of D products, of 64 rows, of one addition and two factors for each chunk (of 32 rows at least), and a weight's exponent off by
  2^-24 of itself (x e^-x <= 0.37): e32 = (2 D + 128 + 4 n / 32) 2^-23 of A or S|.
* weights under fp32's smallest normal number, 2^-126, may be zeros: 2^-120, with terms that are below 64 in all.
* one rounding of the output: u of it, for fp16 2^-25 below 2^-14 (its numbers are 2^-24 apart there, and rounding is off by half of that).

So |o - o64| <= u |o64| + (u + e32) A, for states (4 u^2 + e32) S|, and the same for gradients with the recurrence of theirs.  On the norm, where the
roundings do not conspire: 3 u (|o| large enough for that: a hundred values at least), 1e-5 for fp32.
"""
import math

import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
from tests._harness import TORCH_DT, check_guards, guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return CudaBackend()


def unit(dtype):
    return 0.0 if dtype == "f32" else torch.finfo(TORCH_DT[dtype]).eps / 2


def e32(dim, n):
    return (2 * dim + 128 + n / 8) * 2.0 ** -23


def recurrence(q, k, v, g, scale, first=None):
    """One sequence: q [H, n, K], k [H, n, K], v [H, n, V] (64 bits, heads expanded), g [H]; (out, last state)."""
    lam = torch.exp(g)[:, None, None]
    s = torch.zeros(q.shape[0], q.shape[2], v.shape[2], dtype=q.dtype, device=q.device) if first is None else first
    out = []
    for t in range(q.shape[1]):
        s = lam * s + k[:, t, :, None] * v[:, t, None, :]
        out.append(scale * (q[:, t, None, :] @ s)[:, 0])
    return (torch.stack(out, 1) if out else q.new_zeros(q.shape[0], 0, v.shape[2])), s


def near(got, ref, bound, u, what, norm=None):
    ref = ref.to(got.device)
    assert got.shape == ref.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    ok = ~torch.isnan(ref)
    off = (got.double() - ref).abs()[ok]
    most = (u * ref.abs() + bound)[ok] + (2.0 ** -25 if got.dtype is torch.float16 else 2.0 ** -120)
    assert bool((off <= most).all()), f"{what}: off by {float(off.max()):.3g}, {float((off / most.clamp(min=1e-300)).max()):.3g} of what is allowed"
    if norm is not None and off.numel() >= 100 and float(ref[ok].norm()) > 0:
        assert float(off.norm() / ref[ok].norm()) <= norm, f"{what}: {float(off.norm() / ref[ok].norm()):.3g} on the norm"


def decays(heads, kind):
    h = torch.arange(heads, dtype=torch.float64)
    if kind == "none":
        return None
    if kind == "spread":
        g = -(0.7 ** (1 - h / max(1, heads - 1))) * 2.0 ** (-10 * h / max(1, heads - 1))
    else:   # the ends of the range: none kept, all kept, almost none, few
        g = torch.tensor([-math.inf, 0.0, -120.0, -5.0, -1e-6, -0.03125])[h.long() % 6]
    return g.float().cuda()


class Case:
    """Tensors of a call in one of its layouts, and the rows of each sequence."""

    def __init__(self, dtype, lens, heads, kv, key, value, layout, decay="spread", first=False, seed=0, size=0.5, pad=3):
        self.g = torch.Generator(device="cuda").manual_seed(seed + 977 * key + value + sum(lens))
        self.dtype, self.lens, self.heads, self.kv, self.key, self.value, self.layout = dtype, lens, heads, kv, key, value, layout
        self.batch, self.seq = len(lens), max(max(lens), 1) + (pad if layout in ("lengths", "lengths_token") else 0)
        self.size = size
        self.decay = decays(heads, decay)
        self.starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
        self.rows = self.starts[-1] + pad   # packed: some behind the last sequence
        if layout in ("head", "token"):
            assert min(lens) == max(lens)
        self.q, self.k, self.v, self.do = (self.make(h, d) for h, d in ((heads, key), (kv, key), (kv, value), (heads, value)))
        self.first = torch.randn((self.batch, heads, key, value), generator=self.g, device="cuda") * size if first else None

    def shape(self, heads, d):
        if self.layout == "starts":
            return (self.rows, heads, d)
        return (self.batch, heads, self.seq, d) if self.layout in ("head", "lengths") else (self.batch, self.seq, heads, d)

    def make(self, heads, d):
        x = (torch.randn(self.shape(heads, d), generator=self.g, device="cuda") * self.size).to(TORCH_DT[self.dtype])
        if self.layout != "head" and self.layout != "token":   # what no sequence has may be anything
            keep = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
            for b in range(self.batch):
                self.of(keep, b).fill_(True)
            x[~keep] = float("nan")
        return x

    def of(self, x, b):
        """[heads, n, d] of sequence b."""
        n = self.lens[b]
        if self.layout == "starts":
            return x[self.starts[b]:self.starts[b] + n].transpose(0, 1)
        return x[b, :, :n] if self.layout in ("head", "lengths") else x[b, :n].transpose(0, 1)

    def wide(self, x, b):
        y = self.of(x, b).double()
        return y.repeat_interleave(self.heads // y.shape[0], 0)

    def kw(self):
        whole = lambda x: GpuBuffer(torch.tensor(x, dtype=torch.int32, device="cuda"))  # noqa: E731
        return dict(tokenMajor=self.layout in ("token", "lengths_token"), lengths=whole(self.lens) if "lengths" in self.layout else None,
                    tokenStarts=whole(self.starts) if self.layout == "starts" else None)

    def sizes(self):
        return (self.batch, self.heads, self.kv, self.seq, self.key, self.value)

    def buf(self, x):
        return None if x is None else GpuBuffer(x)

    def log_decay(self):
        return self.decay.double() if self.decay is not None else torch.zeros(self.heads, dtype=torch.float64, device="cuda")

    def check_rest(self, x, flat, what):
        """Rows of padding are zeros, rows of no sequence are as they were (NaN), nothing outside was written."""
        check_guards(flat, what)
        if self.layout == "starts":
            assert bool(torch.isnan(x[self.starts[-1]:]).all()), f"{what}: a row behind the last sequence was written"
        elif "lengths" in self.layout:
            y = x.clone()
            for b in range(self.batch):
                self.of(y, b).zero_()
            assert bool((y == 0).all()), f"{what}: padding is not zeros"


def run_forward(backend, c, scale=0.0, last=False):
    flat, out = guarded(c.shape(c.heads, c.value), TORCH_DT[c.dtype], "cuda")
    sflat, final = guarded((c.batch, c.heads, c.key, c.value), torch.float32, "cuda")
    backend.LinearAttention(c.buf(c.q), c.buf(c.k), c.buf(c.v), GpuBuffer(out), c.buf(c.decay), *c.sizes(), scale, initialStates=c.buf(c.first),
                            finalStates=GpuBuffer(final) if last else None, **c.kw())
    torch.cuda.synchronize()
    c.check_rest(out, flat, "out")
    check_guards(sflat, "final states")
    return out, final


def check_forward(backend, c, last=True):
    out, final = run_forward(backend, c, last=last)
    u, scale = unit(c.dtype), c.key ** -0.5
    round_u = torch.finfo(TORCH_DT[c.dtype]).eps / 2
    for b, n in enumerate(c.lens):
        q, k, v, g = c.wide(c.q, b), c.wide(c.k, b), c.wide(c.v, b), c.log_decay()
        first = c.first[b].double() if c.first is not None else None
        ref, state = recurrence(q, k, v, g, scale, first)
        size, size_s = recurrence(q.abs(), k.abs(), v.abs(), g, scale, None if first is None else first.abs())
        e = e32(max(c.key, c.value), n)
        near(c.of(out, b), ref, (u + e) * size, round_u, f"sequence {b} of {n}", 1e-5 if c.dtype == "f32" else 3 * u)
        if last:
            near(final[b], state, (4 * u * u + e) * size_s, 2.0 ** -24, f"state of sequence {b}", 1e-5)


DIMS = [(64, 64), (128, 128), (64, 128), (128, 64), (32, 32), (40, 72), (256, 256), (8, 16), (96, 40)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("key,value", DIMS)
def test_forward_sizes(backend, dtype, key, value):
    check_forward(backend, Case(dtype, [130, 130], 4, 2, key, value, "head", first=True))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("layout,lens", [("head", [1]), ("token", [64, 64]), ("head", [65]), ("token", [128]), ("head", [63, 63, 63]),
                                         ("lengths", [0, 1, 300, 64]), ("lengths_token", [127, 128, 129]),
                                         ("starts", [5, 0, 200, 1, 64, 65]), ("starts", [0, 0]), ("lengths", [0])])
def test_forward_lengths(backend, dtype, dim, layout, lens):
    check_forward(backend, Case(dtype, lens, 3, 3, dim, dim, layout, first=True, seed=1))
    check_forward(backend, Case(dtype, lens, 2, 1, dim, dim, layout, decay="none", seed=2))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("key,value", [(128, 128), (64, 64), (48, 56)])
def test_forward_decays(backend, dtype, key, value):
    """Heads that keep nothing, everything, almost nothing: no product of a zero and an infinity anywhere."""
    check_forward(backend, Case(dtype, [150, 70], 6, 2, key, value, "starts", decay="ends", first=True, seed=3))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_forward_long(backend, dtype, dim):
    check_forward(backend, Case(dtype, [2111], 4, 4, dim, dim, "head", first=True, seed=4))


@pytest.mark.parametrize("dtype,size", [("f16", 60.0), ("f16", 1.0 / 512), ("bf16", 1e4), ("bf16", 1e-6)])
@pytest.mark.parametrize("dim", [64, 128])
def test_forward_magnitudes(backend, dtype, size, dim):
    """Products and states far outside of fp16's range, and far below its smallest numbers, where the outputs are within it."""
    c = Case(dtype, [200], 2, 2, dim, dim, "head", decay="spread", seed=5, size=size)
    c.q = c.q / size if dtype == "f16" and size > 1 else c.q
    out, _ = run_forward(backend, c)
    q, k, v = (c.wide(x, 0) for x in (c.q, c.k, c.v))
    ref, _ = recurrence(q, k, v, c.log_decay(), dim ** -0.5)
    top, _ = recurrence(q.abs(), k.abs(), v.abs(), c.log_decay(), dim ** -0.5)
    if dtype == "f16":
        ref = torch.where(ref.abs() >= 65520, ref.sign() * math.inf, ref)
    fine = torch.isfinite(ref)
    tiny = 0.0 if dtype == "bf16" else 2.0 ** -25   # half of fp16's smallest number, for the output's rounding
    u = unit(dtype)
    got = c.of(out, 0).double()
    at_edge = (ref.abs() - 65520).abs() <= (2 * u + e32(dim, 200)) * top if dtype == "f16" else torch.zeros_like(fine)
    fine &= ~at_edge
    assert bool(((got - ref).abs()[fine] <= (u * ref.abs() + (u + e32(dim, 200)) * top + tiny)[fine]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 48])
def test_what_follows_a_row_does_not_reach_it(backend, dtype, dim):
    """NaN and infinities in the last rows of keys, values and queries: the rows before them are what they were.  (A kernel may sum a row that shares
    a tile with such a value in another order.  Two fp32 sums of the same 64 products are each off by 64 * 2^-24 of their terms, and with the
    factors behind them differ by 2^-16 A at most; each is rounded once, by u of it.)"""
    c = Case(dtype, [140], 2, 2, dim, dim, "head", seed=6)
    clean, _ = run_forward(backend, c)
    top, _ = recurrence(*(x[0].double().abs() for x in (c.q, c.k, c.v)), c.log_decay(), dim ** -0.5)
    most = 2 * torch.finfo(TORCH_DT[dtype]).eps / 2 * clean.double().abs() + 2.0 ** -16 * top
    for at in (139, 100, 64, 3):
        for bad in (float("nan"), float("inf")):
            q, k, v = c.q.clone(), c.k.clone(), c.v.clone()
            q[:, :, at:] = bad
            k[:, 0, at:, 1::2] = bad
            v[:, 1, at:, ::3] = bad
            keep = c.q, c.k, c.v
            c.q, c.k, c.v = q, k, v
            out, _ = run_forward(backend, c)
            c.q, c.k, c.v = keep
            assert bool(((out.double() - clean.double()).abs() <= most)[:, :, :at].all()), (at, bad)
            assert bool(torch.isnan(out[:, :, at]).any())


def test_a_value_that_is_not_finite_stays_in_its_column(backend):
    """A NaN value makes its column NaN from its row on, and leaves the others."""
    for dtype in ("bf16", "f16", "f32"):
        for dim in (64, 128):
            c = Case(dtype, [200], 1, 1, dim, dim, "head", seed=7)
            clean, _ = run_forward(backend, c)
            c.v[0, 0, 70, 5] = float("nan")
            out, _ = run_forward(backend, c)
            hit = torch.zeros_like(out, dtype=torch.bool)
            hit[0, 0, 70:, 5] = True
            assert torch.equal(torch.isnan(out), hit)
            top, _ = recurrence(*(x[0].double().abs().nan_to_num() for x in (c.q, c.k, c.v)), c.log_decay(), dim ** -0.5)
            most = 2 * torch.finfo(TORCH_DT[dtype]).eps / 2 * clean.double().abs() + 2.0 ** -16 * top   # (as above)
            assert bool(((out.double() - clean.double()).abs() <= most)[~hit].all())


def test_decay_above_zero_or_nan_shows(backend):
    for dtype, dim in (("bf16", 128), ("f32", 32)):
        c = Case(dtype, [70], 3, 3, dim, dim, "head", seed=8)
        c.decay = torch.tensor([0.1, -0.1, math.nan], device="cuda")
        out, _ = run_forward(backend, c)
        assert bool(torch.isnan(out[:, [0, 2]]).all()) and bool(torch.isfinite(out[:, 1]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 24])
def test_state_slots(backend, dtype, dim):
    """Slots in any order, in place; a negative one is no state; one that is not there or has been taken gives NaN and is left alone."""
    lens = [70, 3, 130, 20, 64, 9]
    c = Case(dtype, lens, 2, 2, dim, dim, "starts", seed=9)
    flat, pool = guarded((5, 2, dim, dim), torch.float32, "cuda")
    pool.copy_(torch.randn(5, 2, dim, dim, device="cuda"))
    was = pool.clone()
    slots = [3, -1, 0, 5, 3, 2]
    oflat, out = guarded(c.shape(2, dim), TORCH_DT[dtype], "cuda")
    backend.LinearAttention(c.buf(c.q), c.buf(c.k), c.buf(c.v), GpuBuffer(out), c.buf(c.decay), *c.sizes(), initialStates=GpuBuffer(pool),
                            finalStates=GpuBuffer(pool), stateSlots=GpuBuffer(torch.tensor(slots, dtype=torch.int32, device="cuda")), **c.kw())
    torch.cuda.synchronize()
    check_guards(flat, "pool")
    c.check_rest(out, oflat, "out")
    for b, s in enumerate(slots):
        got = c.of(out, b)
        if b in (3, 4):
            assert bool(torch.isnan(got).all())
            continue
        q, k, v, g = c.wide(c.q, b), c.wide(c.k, b), c.wide(c.v, b), c.log_decay()
        first = was[s].double() if s >= 0 else None
        ref, state = recurrence(q, k, v, g, dim ** -0.5, first)
        size, size_s = recurrence(q.abs(), k.abs(), v.abs(), g, dim ** -0.5, None if first is None else first.abs())
        e, u = e32(dim, lens[b]), unit(dtype)
        near(got, ref, (u + e) * size, torch.finfo(TORCH_DT[dtype]).eps / 2, f"sequence {b}")
        if s >= 0:
            near(pool[s], state, (4 * u * u + e) * size_s, 2.0 ** -24, f"slot {s}")
    for s in (1, 4):
        assert torch.equal(pool[s], was[s])


@pytest.mark.parametrize("dtype,key,value", [("bf16", 128, 128), ("f16", 64, 128), ("bf16", 64, 64), ("f32", 64, 64), ("f32", 40, 72), ("bf16", 96, 40)])
def test_segments(backend, dtype, key, value):
    """Long sequences of few heads are cut into segments that run at once: ragged ones too, with states in and out, in place and through slots; and the
    same call without a workspace, which is not cut."""
    c = Case(dtype, [3000, 1, 0, 2400], 1, 1, key, value, "starts", first=True, seed=20)
    block = dict(batch=4, heads=1, kv_heads=1, seq_len=3000, key_dim=key, value_dim=value, dtype={"bf16": N.BF16, "f16": N.F16, "f32": N.F32}[dtype])
    assert N.linear_workspace_bytes(N.linear_block(**block)) > 0
    check_forward(backend, c)
    pool = torch.randn(6, 1, key, value, device="cuda")
    slots = torch.tensor([4, 0, 5, 1], dtype=torch.int32, device="cuda")
    outs, pools = [], []
    for cut in (True, False):
        now, out = pool.clone(), torch.empty(c.shape(1, value), dtype=TORCH_DT[dtype], device="cuda")
        if cut:
            backend.LinearAttention(c.buf(c.q), c.buf(c.k), c.buf(c.v), GpuBuffer(out), c.buf(c.decay), *c.sizes(), initialStates=GpuBuffer(now),
                                    finalStates=GpuBuffer(now), stateSlots=GpuBuffer(slots), **c.kw())
        else:
            starts = torch.tensor(c.starts, dtype=torch.int32, device="cuda")
            N.linear_attention(N.linear_block(q=c.q.data_ptr(), k=c.k.data_ptr(), v=c.v.data_ptr(), out=out.data_ptr(), decay=c.decay.data_ptr(),
                                              token_starts=starts.data_ptr(), tokens=c.rows, initial_state=now.data_ptr(), final_state=now.data_ptr(),
                                              state_slots=slots.data_ptr(), num_slots=6, **block), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        outs.append(out[:c.starts[-1]].double())
        pools.append(now.double())
    # both are within the bounds of the recurrence, so within twice those of one another
    for b, n in enumerate(c.lens):
        q, k, v = c.wide(c.q, b), c.wide(c.k, b), c.wide(c.v, b)
        size, size_s = recurrence(q.abs(), k.abs(), v.abs(), c.log_decay(), key ** -0.5, pool[slots[b]].double().abs())
        e, u = e32(max(key, value), n), unit(dtype)
        rows = slice(c.starts[b], c.starts[b] + n)
        near(outs[0][rows].transpose(0, 1), outs[1][rows].transpose(0, 1), 2 * (u + e) * size, 2 * torch.finfo(TORCH_DT[dtype]).eps / 2, f"sequence {b}")
        near(pools[0][slots[b]], pools[1][slots[b]], 2 * (4 * u * u + e) * size_s, 2.0 ** -23, f"state of sequence {b}")
    assert torch.equal(pools[0][[2, 3]], pool.double()[[2, 3]])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows_at_all(backend, dtype):
    """A packed batch of empty sequences: the states go through as they are, forwards and backwards (times one step's decay to the power of no rows)."""
    empty = lambda h: GpuBuffer(torch.empty(0, h, 64, dtype=TORCH_DT[dtype], device="cuda"))  # noqa: E731
    first, last, grad, back = torch.randn(2, 4, 64, 64, device="cuda"), *(torch.zeros(2, 4, 64, 64, device="cuda") for _ in range(3))
    grad.copy_(first.flip(0))
    starts = GpuBuffer(torch.zeros(3, dtype=torch.int32, device="cuda"))
    decay = decays(4, "spread")
    sizes = (2, 4, 2, 8, 64, 64)
    backend.LinearAttention(empty(4), empty(2), empty(2), empty(4), GpuBuffer(decay), *sizes, tokenStarts=starts, initialStates=GpuBuffer(first),
                            finalStates=GpuBuffer(last))
    backend.LinearAttentionBackward(empty(4), empty(4), empty(2), empty(2), empty(4), empty(2), empty(2), GpuBuffer(decay), *sizes, tokenStarts=starts,
                                    initialStates=GpuBuffer(first), gradFinalStates=GpuBuffer(grad), gradInitialStates=GpuBuffer(back))
    torch.cuda.synchronize()
    assert torch.equal(last, first) and torch.equal(back, grad)


@pytest.mark.parametrize("key,value", [(128, 128), (64, 128), (72, 40)])
def test_segments_backward(backend, key, value):
    check_backward(backend, Case("bf16", [2300, 5, 1900], 1, 1, key, value, "lengths_token", first=True, seed=21), last=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tensors_that_no_tile_load_fits(backend, dtype):
    """Strides of odd numbers of elements, a shared row (stride 0) and unaligned addresses, through the C ABI: other kernels, the same results."""
    n, heads, dim = 70, 2, 64
    g = torch.Generator(device="cuda").manual_seed(22)
    make = lambda: (torch.randn(20000, generator=g, device="cuda") * 0.5).to(TORCH_DT[dtype])  # noqa: E731
    q = torch.as_strided(make(), (heads, n, dim), (67, 135, 1), 1)
    k = torch.as_strided(make(), (heads, n, dim), (0, 64, 1), 8)          # one head's keys for both
    v = torch.as_strided(make(), (heads, n, dim), (4800, 66, 1), 0)
    to = torch.zeros(20000, dtype=q.dtype, device="cuda")
    out = torch.as_strided(to, (heads, n, dim), (65, 133, 1), 3)
    decay = decays(heads, "spread")
    N.linear_attention(N.linear_block(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), decay=decay.data_ptr(), batch=1, heads=heads,
                                      kv_heads=heads, seq_len=n, key_dim=dim, value_dim=dim, dtype=N.BF16 if dtype == "bf16" else N.F16,
                                      q_stride=(0, 67, 135), k_stride=(0, 0, 64), v_stride=(0, 4800, 66), o_stride=(0, 65, 133)),
                       torch.cuda.current_stream().cuda_stream)
    ins = [x.double() for x in (q, k, v)]
    ref, _ = recurrence(*ins, decay.double(), dim ** -0.5)
    size, _ = recurrence(*(x.abs() for x in ins), decay.double(), dim ** -0.5)
    near(out, ref, (unit(dtype) + e32(dim, n)) * size, torch.finfo(TORCH_DT[dtype]).eps / 2, "out")


# ---- gradients -------------------------------------------------------------------------------------------------------

def run_backward(backend, c, d_last=None, want_first=False):
    made = {n: guarded(c.shape(h, d), TORCH_DT[c.dtype], "cuda") for n, h, d in (("dq", c.heads, c.key), ("dk", c.kv, c.key), ("dv", c.kv, c.value))}
    sflat, d_first = guarded((c.batch, c.heads, c.key, c.value), torch.float32, "cuda")
    backend.LinearAttentionBackward(c.buf(c.do), c.buf(c.q), c.buf(c.k), c.buf(c.v), *(GpuBuffer(made[n][1]) for n in ("dq", "dk", "dv")),
                                    c.buf(c.decay), *c.sizes(), initialStates=c.buf(c.first), gradFinalStates=c.buf(d_last),
                                    gradInitialStates=GpuBuffer(d_first) if want_first else None, **c.kw())
    torch.cuda.synchronize()
    for n, (flat, x) in made.items():
        c.check_rest(x, flat, n)
    check_guards(sflat, "gradient of first states")
    return {n: x for n, (_, x) in made.items()}, d_first


def gradients(q, k, v, do, g, scale, first, d_last, group):
    """64 bits, by the recurrence's own derivative; heads of k and v summed."""
    q, k, v = (x.detach().clone().requires_grad_(True) for x in (q, k, v))
    s0 = (first if first is not None else q.new_zeros(q.shape[0], q.shape[2], v.shape[2])).detach().clone().requires_grad_(True)
    out, last = recurrence(q, k, v, g, scale, s0)
    total = (out * do).sum() + ((last * d_last).sum() if d_last is not None else 0 * last.sum())
    dq, dk, dv, ds = torch.autograd.grad(total, (q, k, v, s0), allow_unused=True)
    zero = lambda d, x: torch.zeros_like(x) if d is None else d  # noqa: E731
    dq, dk, dv, ds = zero(dq, q), zero(dk, k), zero(dv, v), zero(ds, s0)
    share = lambda x: x.unflatten(0, (-1, group)).sum(1)  # noqa: E731
    return dq, share(dk), share(dv), ds


def check_backward(backend, c, last=False):
    d_last = torch.randn((c.batch, c.heads, c.key, c.value), generator=c.g, device="cuda") * c.size if last else None
    got, d_first = run_backward(backend, c, d_last, True)
    u, scale, group = unit(c.dtype), c.key ** -0.5, c.heads // c.kv
    round_u = torch.finfo(TORCH_DT[c.dtype]).eps / 2
    for b, n in enumerate(c.lens):
        ins = [c.wide(x, b) for x in (c.q, c.k, c.v, c.do)]
        first, end = (None if x is None else x[b].double() for x in (c.first, d_last))
        ref = gradients(*ins, c.log_decay(), scale, first, end, group)
        size = gradients(*(x.abs() for x in ins), c.log_decay(), scale, None if first is None else first.abs(), None if end is None else end.abs(), group)
        e = e32(max(c.key, c.value), n)
        for i, name in enumerate(("dq", "dk", "dv")):
            near(c.of(got[name], b), ref[i], (u + e) * size[i], round_u, f"{name} of sequence {b} of {n}", 1e-5 if c.dtype == "f32" else 3 * u)
        near(d_first[b], ref[3], (4 * u * u + e) * size[3], 2.0 ** -24, f"gradient of first state {b}", 1e-5)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("key,value", DIMS)
def test_backward_sizes(backend, dtype, key, value):
    check_backward(backend, Case(dtype, [130, 130], 4, 2, key, value, "head", first=True), last=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("layout,lens", [("head", [1]), ("token", [64, 64]), ("head", [65]), ("lengths", [0, 1, 200, 64]),
                                         ("lengths_token", [127, 128, 129]), ("starts", [5, 0, 200, 1, 64, 65]), ("starts", [0, 0])])
def test_backward_lengths(backend, dtype, dim, layout, lens):
    check_backward(backend, Case(dtype, lens, 3, 3, dim, dim, layout, first=True, seed=1), last=True)
    check_backward(backend, Case(dtype, lens, 6, 2, dim, dim, layout, decay="none", seed=2))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("key,value", [(128, 128), (64, 64), (48, 56)])
def test_backward_decays(backend, dtype, key, value):
    check_backward(backend, Case(dtype, [150, 70], 6, 2, key, value, "starts", decay="ends", first=True, seed=3), last=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_long(backend, dtype):
    check_backward(backend, Case(dtype, [1100], 2, 2, 128, 128, "head", first=True, seed=4), last=True)


@pytest.mark.parametrize("dim", [64, 40])
def test_backward_against_differences(backend, dim):
    """The loss is linear in each input by itself, so that a difference over any step is its gradient times the step: in fp32,
    (loss(x + d) - loss(x)) against <gradient, d>, each a sum whose terms are off by e32 of them."""
    c = Case("f32", [90, 90], 4, 2, dim, dim, "token", first=True, seed=10)
    got, d_first = run_backward(backend, c, None, True)

    def loss():
        out, _ = run_forward(backend, c)
        return (out.double() * c.do.double()).sum(), (out.double().abs() * c.do.double().abs()).sum()

    base, size = loss()
    e = e32(dim, 90)
    for name, grad in (("q", got["dq"]), ("k", got["dk"]), ("v", got["dv"]), ("first", d_first)):
        x = getattr(c, name)
        d = torch.randn_like(x)
        moved = x + d
        setattr(c, name, moved)
        there, size2 = loss()
        setattr(c, name, x)
        d = moved.double() - x.double()   # the step as it was taken
        # (terms of the sums behind an output are larger than it by the square root of their number, 90 * dim at most)
        assert abs(float(there - base - (grad.double() * d).sum())) <= 4 * e * math.sqrt(90 * dim) * float(size + size2), name


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_is_the_same_twice(backend, dtype):
    """No atomics: bit for bit, shared heads too."""
    c = Case(dtype, [300, 77], 8, 2, 64, 64, "starts", first=True, seed=11)
    a, sa = run_backward(backend, c, None, True)
    b, sb = run_backward(backend, c, None, True)
    for n in a:
        assert torch.equal(a[n].view(torch.uint8), b[n].view(torch.uint8))
    assert torch.equal(sa, sb)


# ---- single tokens ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("batch,heads,kv,key,value", [(1, 32, 32, 128, 128), (3, 4, 2, 64, 128), (5, 6, 1, 40, 72), (2, 2, 2, 256, 256), (70, 3, 3, 64, 64),
                                                      (1, 1, 1, 8, 8), (2, 5, 5, 96, 40), (300, 1, 1, 32, 16)])
def test_step(backend, dtype, batch, heads, kv, key, value):
    g = torch.Generator(device="cuda").manual_seed(batch + key)
    make = lambda *s: (torch.randn(s, generator=g, device="cuda") * 0.5).to(TORCH_DT[dtype])  # noqa: E731
    q, k, v = make(batch, heads, key), make(batch, kv, key), make(batch, kv, value)
    flat, pool = guarded((batch + 2, heads, key, value), torch.float32, "cuda")
    pool.copy_(torch.randn(pool.shape, generator=g, device="cuda"))
    was, oflat_out = pool.clone(), guarded((batch, heads, value), TORCH_DT[dtype], "cuda")
    slots = torch.randperm(batch + 2, generator=g, device="cuda")[:batch].to(torch.int32)
    decay = decays(heads, "ends")
    backend.LinearAttentionStep(GpuBuffer(q), GpuBuffer(k), GpuBuffer(v), GpuBuffer(oflat_out[1]), GpuBuffer(pool), GpuBuffer(decay), batch, heads,
                                kv, key, value, stateSlots=GpuBuffer(slots))
    torch.cuda.synchronize()
    check_guards(flat, "pool")
    check_guards(oflat_out[0], "out")
    wide = lambda x: x.double().repeat_interleave(heads // x.shape[1], 1)  # noqa: E731
    first = was[slots.long()].double()
    lam, kk, vv = torch.exp(decay.double())[:, None, None], wide(k), wide(v)
    state = lam * first + kk[..., :, None] * vv[..., None, :]
    size_s = lam * first.abs() + kk.abs()[..., :, None] * vv.abs()[..., None, :]
    ref = (q.double()[..., None, :] @ state)[..., 0, :] * key ** -0.5
    size = (q.double().abs()[..., None, :] @ size_s)[..., 0, :] * key ** -0.5
    near(pool[slots.long()], state, 2.0 ** -21 * size_s, 2.0 ** -24, "states")
    near(oflat_out[1], ref, e32(key, 1) * size, torch.finfo(TORCH_DT[dtype]).eps / 2, "out")
    rest = torch.ones(batch + 2, dtype=torch.bool, device="cuda")
    rest[slots.long()] = False
    assert torch.equal(pool[rest], was[rest])


def test_step_slots(backend):
    """Padding rows, a slot that is not there, one that an earlier row has."""
    q, k, v = (torch.randn(6, 2, 64, device="cuda").half() for _ in range(3))
    pool = torch.randn(4, 2, 64, 64, device="cuda")
    was, out = pool.clone(), torch.full((6, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    slots = torch.tensor([2, -1, 4, 0, 2, -5], dtype=torch.int32, device="cuda")
    backend.LinearAttentionStep(GpuBuffer(q), GpuBuffer(k), GpuBuffer(v), GpuBuffer(out), GpuBuffer(pool), None, 6, 2, 2, 64, 64,
                                stateSlots=GpuBuffer(slots))
    assert bool((out[[1, 5]] == 0).all()) and bool(torch.isnan(out[[2, 4]]).all()) and bool(torch.isfinite(out[[0, 3]]).all())
    assert torch.equal(pool[[1, 3]], was[[1, 3]])
    for b, s in ((0, 2), (3, 0)):
        near(pool[s], was[s].double() + k[b].double()[..., :, None] * v[b].double()[..., None, :], 2.0 ** -22 * was[s].double().abs().clamp(min=1), 2.0 ** -24, "state")


def test_step_rows_at_any_distance(backend):
    """Rows of a packed projection, through the C ABI: nothing but the elements' own alignment."""
    x = torch.randn(3 * 601 + 5, device="cuda").bfloat16()
    at = lambda off: torch.as_strided(x, (3, 4, 40), (601, 43, 1), off)  # noqa: E731
    q, k, v, out = at(1), at(174), at(347), torch.zeros(3, 4, 40, device="cuda").bfloat16()
    pool = torch.zeros(3, 4, 40, 40, device="cuda")
    N.linear_attention_step(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), states=pool.data_ptr(), batch=3, heads=4, kv_heads=4,
                            key_dim=40, value_dim=40, dtype=N.BF16, stream=torch.cuda.current_stream().cuda_stream, q_stride=(601, 43),
                            k_stride=(601, 43), v_stride=(601, 43), scale=0.25)
    ref = 0.25 * (q.double() * k.double()).sum(-1, keepdim=True) * v.double()
    size = 0.25 * (q.double() * k.double()).abs().sum(-1, keepdim=True) * v.double().abs()
    near(out, ref, e32(40, 1) * size, 2.0 ** -9 * 2, "out")


# ---- the operators together ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [128, 48])
def test_prompt_then_tokens_is_the_prompt_at_once(backend, dtype, dim):
    """A prompt of n tokens that leaves its states, and m steps that go on from them, against one prompt of n + m: the states' rounding where they
    meet queries is the only difference, within the bounds of both."""
    n, m, heads = 75, 6, 4
    c = Case(dtype, [n + m], heads, 2, dim, dim, "token", seed=12)
    whole, last = run_forward(backend, c, last=True)
    pool, out = torch.zeros(3, heads, dim, dim, device="cuda"), torch.empty(n, heads, dim, dtype=TORCH_DT[dtype], device="cuda")
    slot = GpuBuffer(torch.tensor([1], dtype=torch.int32, device="cuda"))
    part = lambda x, a, b: GpuBuffer(x[0, a:b].contiguous())  # noqa: E731
    backend.LinearAttention(part(c.q, 0, n), part(c.k, 0, n), part(c.v, 0, n), GpuBuffer(out), c.buf(c.decay), 1, heads, 2, n, dim, dim, tokenMajor=True,
                            initialStates=GpuBuffer(pool), finalStates=GpuBuffer(pool), stateSlots=slot)
    rows = [out]
    for t in range(n, n + m):
        o = torch.empty(1, heads, dim, dtype=TORCH_DT[dtype], device="cuda")
        backend.LinearAttentionStep(part(c.q, t, t + 1), part(c.k, t, t + 1), part(c.v, t, t + 1), GpuBuffer(o), GpuBuffer(pool), c.buf(c.decay), 1, heads,
                                    2, dim, dim, stateSlots=slot)
        rows.append(o)
    q, k, v = (c.wide(x, 0) for x in (c.q, c.k, c.v))
    size, size_s = recurrence(q.abs(), k.abs(), v.abs(), c.log_decay(), dim ** -0.5)
    u, e = unit(dtype), e32(dim, n + m)
    near(torch.cat(rows).transpose(0, 1), whole[0].double().transpose(0, 1), 2 * (u + e) * size, 2 * torch.finfo(TORCH_DT[dtype]).eps / 2, "outputs")
    near(pool[1], last[0].double(), 2 * (4 * u * u + e) * size_s, 2.0 ** -23, "states")
    assert bool((pool[[0, 2]] == 0).all())


def test_layer_with_rotated_heads(backend):
    """Rotary positions in front of linear attention, forwards and backwards, against autograd of both in 64 bits."""
    n, heads, kv, dim, part = 100, 4, 2, 64, 32
    c = Case("f32", [n], heads, kv, dim, dim, "token", seed=13)
    f = backend.RotaryFrequencies(part, scaling="parts", factor=4.0, originalLength=64)
    q, k = torch.empty_like(c.q), torch.empty_like(c.k)
    args = (f, n, heads, kv, dim)
    backend.RotaryEmbedding(c.buf(c.q), GpuBuffer(q), c.buf(c.k), GpuBuffer(k), *args, interleaved=False)
    raw = c.q, c.k
    c.q, c.k = q, k
    out, _ = run_forward(backend, c)
    got, _ = run_backward(backend, c)
    gq, gk = torch.empty_like(q), torch.empty_like(k)
    backend.RotaryEmbeddingBackward(GpuBuffer(got["dq"]), GpuBuffer(gq), GpuBuffer(got["dk"]), GpuBuffer(gk), *args, interleaved=False)
    x, y, v = (t[0].double().transpose(0, 1).clone().requires_grad_(True) for t in (*raw, c.v))
    angle = torch.arange(n, device="cuda").double()[:, None] * f.tensor
    turn = lambda t: torch.cat((t[..., :16] * angle.cos() - t[..., 16:32] * angle.sin(), t[..., :16] * angle.sin() + t[..., 16:32] * angle.cos(), t[..., 32:]), -1)  # noqa: E731
    wide = lambda t: t.repeat_interleave(heads // kv, 0)  # noqa: E731
    ref, _ = recurrence(turn(x), wide(turn(y)), wide(v), c.log_decay(), dim ** -0.5)
    grads = torch.autograd.grad((ref * c.do[0].double().transpose(0, 1)).sum(), (x, y, v))
    for a, b in zip((out, gq, gk, got["dv"]), (ref.detach(), *grads)):
        assert float((a[0].double().transpose(0, 1) - b).norm() / b.norm()) <= 1e-5


@pytest.mark.parametrize("dim", [64, 128])
def test_waits_that_run_out_are_reported(backend, dim):
    """The kernel with bounded waits, its loads withheld: it ends, says so once, and the next call is right."""
    c = Case("bf16", [300], 2, 2, dim, dim, "head", seed=17)
    clean, _ = run_forward(backend, c)
    stream = torch.cuda.current_stream().cuda_stream
    N.linear_attention_poll(stream)
    assert N.load().aidn_sdpa_debug_set(None, None, 5) == N.OK
    run_forward(backend, c)
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_poll(stream)
    assert e.value.status == N.ETIMEOUT
    N.linear_attention_poll(stream)
    assert torch.equal(run_forward(backend, c)[0], clean)


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 40)])
def test_captured_and_replayed(backend, dtype, dim):
    """Forward, backward and step in one graph, on a stream of its own: replays on new inputs give what eager calls give."""
    stream = torch.cuda.Stream()
    own = CudaBackend(stream=stream)
    c = Case(dtype, [100, 70], 4, 2, dim, dim, "starts", seed=14)
    kw = c.kw()
    out = torch.zeros(c.shape(4, dim), dtype=TORCH_DT[dtype], device="cuda")
    grads = [torch.zeros(c.shape(h, dim), dtype=out.dtype, device="cuda") for h in (4, 2, 2)]
    states, o1 = torch.zeros(2, 4, dim, dim, device="cuda"), torch.zeros(2, 4, dim, dtype=out.dtype, device="cuda")
    tok = [x[:2].clone().nan_to_num() for x in (c.q, c.k, c.v)]

    def calls(b):
        b.LinearAttention(c.buf(c.q), c.buf(c.k), c.buf(c.v), GpuBuffer(out), c.buf(c.decay), *c.sizes(), finalStates=GpuBuffer(states), **kw)
        b.LinearAttentionBackward(c.buf(c.do), c.buf(c.q), c.buf(c.k), c.buf(c.v), *(GpuBuffer(g) for g in grads), c.buf(c.decay), *c.sizes(), **kw)
        b.LinearAttentionStep(*(GpuBuffer(x) for x in tok), GpuBuffer(o1), GpuBuffer(states), c.buf(c.decay), 2, 4, 2, dim, dim)

    torch.cuda.synchronize()
    calls(own)   # (the first call of a kernel raises its limits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls(own)
    for x in (c.q, c.k, c.v, c.do):
        x[:c.starts[-1]] = torch.randn(x[:c.starts[-1]].shape, device="cuda")
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (out, *grads, states, o1)]
    calls(backend)
    torch.cuda.synchronize()
    for a, b in zip(got, (out, *grads, states, o1)):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    del graph


def test_two_streams_at_once(backend):
    """Calls of one backend each on two streams, with workspaces of their own."""
    cases = [Case("bf16", [700], 8, 2, 128, 128, "head", seed=s) for s in (15, 16)]
    streams = [torch.cuda.Stream() for _ in cases]
    backends = [CudaBackend(stream=s) for s in streams]
    alone = [run_backward(backend, c)[0] for c in cases]
    made = [[torch.zeros(c.shape(h, 128), dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2)] for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, c, m in zip(backends, cases, made):
            b.LinearAttentionBackward(c.buf(c.do), c.buf(c.q), c.buf(c.k), c.buf(c.v), *(GpuBuffer(g) for g in m), c.buf(c.decay), *c.sizes())
    torch.cuda.synchronize()
    for a, m in zip(alone, made):
        for n, x in zip(("dq", "dk", "dv"), m):
            assert torch.equal(a[n], x)


def test_refusals(backend):
    c = Case("f32", [8], 4, 2, 64, 64, "head")
    out = torch.zeros(c.shape(4, 64), device="cuda")
    state = GpuBuffer(torch.zeros(1, 4, 64, 64, device="cuda"))
    good = dict(query=c.buf(c.q), key=c.buf(c.k), value=c.buf(c.v), output=GpuBuffer(out), decay=c.buf(c.decay), batch=1, heads=4, kvHeads=2, seqLen=8,
                keyDim=64, valueDim=64)
    half = GpuBuffer(torch.zeros(1, 4, 8, 64, device="cuda").half())
    small = GpuBuffer(torch.zeros(1, 4, 8, 32, device="cuda"))
    whole = lambda *v: GpuBuffer(torch.tensor(v, dtype=torch.int32, device="cuda"))  # noqa: E731
    backend.LinearAttention(**good)
    for change in (dict(seqLen=9), dict(batch=0), dict(kvHeads=3), dict(key=half), dict(output=half), dict(output=small), dict(decay=small, heads=0),
                   dict(decay=half), dict(lengths=GpuBuffer(torch.zeros(1, device="cuda"))), dict(lengths=whole(3), tokenStarts=whole(0, 3)),
                   dict(tokenStarts=whole(0)), dict(initialStates=small), dict(finalStates=half), dict(stateSlots=GpuBuffer(torch.zeros(1, device="cuda")))):
        with pytest.raises(ValueError):
            backend.LinearAttention(**{**good, **change})
    with pytest.raises(N.AidnError):
        backend.LinearAttention(**{**good, "keyDim": 60})
    grads = dict(gradOutput=GpuBuffer(out), gradQuery=GpuBuffer(torch.zeros_like(c.q)), gradKey=GpuBuffer(torch.zeros_like(c.k)), gradValue=GpuBuffer(torch.zeros_like(c.v)))
    back = {k: v for k, v in good.items() if k != "output"} | grads
    backend.LinearAttentionBackward(**back)
    for change in (dict(gradKey=small, seqLen=8, heads=4, kvHeads=4), dict(gradOutput=half), dict(gradInitialStates=small), dict(gradQuery=half)):
        with pytest.raises(ValueError):
            backend.LinearAttentionBackward(**{**back, **change})
    one = {n: GpuBuffer(x[:, :, 0].contiguous()) for n, x in (("query", c.q), ("key", c.k), ("value", c.v), ("output", out))}
    step = dict(**one, states=state, decay=c.buf(c.decay), batch=1, heads=4, kvHeads=2, keyDim=64, valueDim=64)
    backend.LinearAttentionStep(**step)
    for change in (dict(batch=2), dict(batch=-1), dict(kvHeads=3), dict(states=half), dict(states=small), dict(query=half), dict(decay=half),
                   dict(stateSlots=GpuBuffer(torch.zeros(1, device="cuda")))):
        with pytest.raises(ValueError):
            backend.LinearAttentionStep(**{**step, **change})
