"""Rotary positions against the formula in 64 bits.

A turn's error: the angle is reduced in 64 bits and then held in 32 bits as turns of at most 1/2, off by 2^-26 turns or 2^-23.3 radians;
sine and cosine are off by 2^-23 more (two units in the last place of values up to 1), and times the amplitude m by 2^-24 m.  Two products and a sum in
32 bits add 3 * 2^-24 of m (|a| + |b|).  In all 2^-21 m (|a| + |b|) at most, and one rounding to the type.
"""
import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
from tests._harness import AIDN_DT, TORCH_DT, check_guards, guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return CudaBackend()


def formula(x, f, pos, interleaved, amplitude, inverse=False):
    """(result, bound of the parts' magnitudes) in 64 bits: x [tokens, heads, dim]."""
    x, part = x.double(), 2 * f.numel()
    angle = pos.double()[:, None] * f * (-1 if inverse else 1)
    c, s = angle.cos()[:, None] * amplitude, angle.sin()[:, None] * amplitude
    y, size = x.clone(), torch.zeros_like(x)
    at, bt = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = x[..., at], x[..., bt]
    y[..., at], y[..., bt] = a * c - b * s, a * s + b * c
    size[..., at] = size[..., bt] = abs(amplitude) * (a.abs() + b.abs())
    return y, size


def check(got, ref, size, dtype):
    u = torch.finfo(TORCH_DT[dtype]).eps / 2
    off = (got.double() - ref).abs()
    assert bool((off <= u * ref.abs() + 2.0 ** -21 * size).all()), float((off - u * ref.abs() - 2.0 ** -21 * size).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,kv,dim,part,start", [
    (1, 32, 8, 128, 128, 1000003), (3, 4, 4, 64, 64, 0), (257, 2, 1, 64, 32, 5), (33, 3, 0, 96, 24, 70000), (18, 5, 5, 256, 256, 1 << 30),
    (7, 1, 2, 40, 2, 9), (5, 2, 2, 8, 6, 1), (130, 7, 1, 80, 40, 3)])
def test_turned_and_turned_back(backend, dtype, interleaved, tokens, heads, kv, dim, part, start):
    g = torch.Generator(device="cuda").manual_seed(tokens * dim + part)
    q = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(TORCH_DT[dtype])
    k = torch.randn((tokens, kv, dim), generator=g, device="cuda").to(TORCH_DT[dtype]) if kv else None
    f = backend.RotaryFrequencies(part)
    pos = start + torch.arange(tokens, device="cuda")
    (qf, qo), (kf, ko) = guarded(q.shape, q.dtype, "cuda"), guarded((tokens, max(kv, 1), dim), q.dtype, "cuda")
    for inverse, call in ((False, backend.RotaryEmbedding), (True, backend.RotaryEmbeddingBackward)):
        call(GpuBuffer(q), GpuBuffer(qo), GpuBuffer(k) if kv else None, GpuBuffer(ko) if kv else None, f, tokens, heads, kv, dim,
             startPosition=start, interleaved=interleaved, amplitude=1.25)
        for x, y in ((q, qo), (k, ko)):
            if x is not None:
                check(y, *formula(x, f.tensor, pos, interleaved, 1.25, inverse), dtype)
                assert torch.equal(y[..., part:], x[..., part:])
        check_guards(qf, "queries")
        check_guards(kf, "keys")


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_positions_of_any_order(backend, wide):
    far = 1 << 40 if wide is torch.int64 else (1 << 31) - 1
    pos = torch.tensor([5, 0, far, 17, far - 1, -3], dtype=wide, device="cuda")
    x = torch.randn(6, 3, 64, device="cuda")
    y, f = torch.empty_like(x), backend.RotaryFrequencies(64)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(y), None, None, f, 6, 3, 0, 64, positions=GpuBuffer(pos))
    # at 2^40 the 64-bit product itself is off by 2^-13 of a radian or so: the frequency's rounding, which the formula shares; the factor
    # 1 / 2 pi rounds once more, by 2^-53 of 2^37.4 turns (2^-13 radians)
    ref, size = formula(x, f.tensor, pos, True, 1.0)
    slack = torch.where(pos.abs() > 1 << 31, 2.0 ** -11, 2.0 ** -21)[:, None, None]
    assert bool(((y.double() - ref).abs() <= 2.0 ** -24 * ref.abs() + slack * size).all())


def test_batches_repeat_positions(backend):
    x = torch.randn(3 * 37, 2, 64, device="cuda").bfloat16()
    y, f = torch.empty_like(x), backend.RotaryFrequencies(64, scaling="linear", factor=4.0)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(y), None, None, f, 111, 2, 0, 64, seqLen=37, startPosition=11)
    check(y, *formula(x, f.tensor, 11 + torch.arange(111, device="cuda") % 37, True, 1.0), "bf16")


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("part", [128, 32])
def test_packed_rows_and_in_place(backend, interleaved, part):
    """Queries and keys side by side in a packed projection, out of place and in place: values stay as they are."""
    x = torch.randn(19, 8 + 2 * 2, 128, device="cuda").half()
    out, f, pos = torch.empty(19, 10, 128, dtype=x.dtype, device="cuda"), backend.RotaryFrequencies(part), torch.arange(19, device="cuda")
    row = (12 * 128, 128)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(out), None, None, f, 19, 10, 0, 128, interleaved=interleaved, queryStride=row)
    check(out, *formula(x[:, :10], f.tensor, pos, interleaved, 1.0), "f16")
    y = x.clone()
    backend.RotaryEmbedding(GpuBuffer(y), GpuBuffer(y), None, None, f, 19, 10, 0, 128, interleaved=interleaved, queryStride=row)
    assert torch.equal(y[:, :10], out) and torch.equal(y[:, 10:], x[:, 10:])


def test_rows_that_no_vector_fits(backend):
    """Rows and heads at odd distances, through the C ABI."""
    store, to = torch.randn(9 * 301, device="cuda").half(), torch.zeros(9 * 333, device="cuda").half()
    f = backend.RotaryFrequencies(64)
    x, y = torch.as_strided(store, (9, 4, 64), (301, 67, 1), 1), torch.as_strided(to, (9, 4, 64), (333, 71, 1), 3)
    N.rotary(query=x.data_ptr(), query_out=y.data_ptr(), frequencies=f.Handle, tokens=9, heads=4, head_dim=64, rotary_dim=64, dtype=N.F16,
             stream=torch.cuda.current_stream().cuda_stream, layout=N.ROPE_HALVES, query_stride=(301, 67), query_out_stride=(333, 71))
    check(y, *formula(x, f.tensor, torch.arange(9, device="cuda"), False, 1.0), "f16")


def test_gradient_is_the_transpose(backend):
    """<turn(x), g> = <x, turn back(g)>: both sides are sums of n products whose terms are off by 2^-20 of them."""
    x, g = torch.randn(41, 6, 64, device="cuda"), torch.randn(41, 6, 64, device="cuda")
    y, d, f = torch.empty_like(x), torch.empty_like(x), backend.RotaryFrequencies(48)
    for interleaved in (True, False):
        args = (f, 41, 6, 0, 64)
        backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(y), None, None, *args, interleaved=interleaved, amplitude=1.5)
        backend.RotaryEmbeddingBackward(GpuBuffer(g), GpuBuffer(d), None, None, *args, interleaved=interleaved, amplitude=1.5)
        a, b = (y.double() * g.double()).sum(), (x.double() * d.double()).sum()
        assert abs(float(a - b)) <= 2.0 ** -19 * float((y.abs() * g.abs()).double().sum() + (x.abs() * d.abs()).double().sum())


def test_agrees_with_the_interleaved_tables(backend):
    """The fp32 call that takes tables: tables from the same frequencies give the same to 32 bits."""
    x, f = torch.randn(50, 64, device="cuda"), backend.RotaryFrequencies(64)
    angle = torch.arange(60, device="cuda").double()[:, None] * f.tensor
    cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    a, b = torch.empty_like(x), torch.empty_like(x)
    backend.RopeInterleaved(GpuBuffer(x), GpuBuffer(cos), GpuBuffer(sin), GpuBuffer(a), 50, 64, 25, 7)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(b), None, None, f, 50, 1, 0, 64, seqLen=25, startPosition=7)
    bound = 2.0 ** -20 * (x.view(50, 32, 2).abs().sum(-1, keepdim=True).expand(50, 32, 2).reshape(50, 64))
    assert bool(((a - b).abs() <= bound).all())


def test_graph_and_stream(backend):
    """A captured call replayed on new inputs, on a stream of its own."""
    stream = torch.cuda.Stream()
    x, y = torch.randn(12, 4, 64, device="cuda").bfloat16(), torch.zeros(12, 4, 64, device="cuda").bfloat16()
    f, own = backend.RotaryFrequencies(64), CudaBackend(stream=stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.RotaryEmbedding(GpuBuffer(x), GpuBuffer(y), None, None, f, 12, 4, 0, 64)
    x.copy_(torch.randn(12, 4, 64, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    check(y, *formula(x, f.tensor, torch.arange(12, device="cuda"), True, 1.0), "bf16")


def test_refusals(backend):
    x, f = GpuBuffer(torch.zeros(4, 2, 64, device="cuda")), backend.RotaryFrequencies(64)
    good = dict(query=x, queryOut=x, key=None, keyOut=None, frequencies=f, tokens=4, heads=2, kvHeads=0, headDim=64)
    for change in (dict(tokens=5), dict(tokens=-1), dict(heads=0), dict(key=x, keyOut=x), dict(kvHeads=2), dict(queryStride=(129, 64)),
                   dict(frequencies=GpuBuffer(torch.zeros(32, device="cuda"))), dict(positions=GpuBuffer(torch.zeros(4, device="cuda"))),
                   dict(positions=GpuBuffer(torch.zeros(3, dtype=torch.int32, device="cuda"))),
                   dict(queryOut=GpuBuffer(torch.zeros(4, 2, 64, device="cuda").half())),
                   dict(queryOut=GpuBuffer(torch.zeros(4, 2, 32, device="cuda")))):
        with pytest.raises(ValueError):
            backend.RotaryEmbedding(**{**good, **change})
    with pytest.raises(N.AidnError):   # wider than the head
        backend.RotaryEmbedding(**{**good, "frequencies": backend.RotaryFrequencies(66)})
    assert AIDN_DT["f32"] == N.F32
