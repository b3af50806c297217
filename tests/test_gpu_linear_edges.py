"""Rotary positions and linear attention at the edges of its types, sizes and calls.  Bounds not named here are those of test_gpu_linear."""
import math
import os
import subprocess
import sys
from fractions import Fraction

import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
from tests._harness import TORCH_DT, check_guards, guarded
from tests.test_gpu_linear import Case, check_backward, check_forward, e32, near, recurrence
from tests.test_gpu_rotary import check as check_turned
from tests.test_gpu_rotary import formula

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return CudaBackend()


# ---- fp16 values that are small, or weighted to little ---------------------------------------------------------------

def one_row(dim, n, row, size, others, seed):
    """fp16 [1, 1, n, dim]: N(0, size) in one row; the others hold as much, or zeros."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((1, 1, n, dim), generator=g, device="cuda") * size).half()
    keep = x.clone()
    if not others:
        x.zero_()
    x[:, :, row] = keep[:, :, row]
    return x


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [64, 50])
@pytest.mark.parametrize("decay,size", [(math.log(0.7), 1.3e-6), (-0.7, 1.0), (-0.7, 1e-6), (-0.1, 60.0)])
@pytest.mark.parametrize("back", [False, True])
def test_small_fp16_values_in_states(backend, dim, n, decay, size, back):
    """What one row adds to a state of a chunk: S = w k v^T (w = exp(decay * rows behind it)), and for the gradient of a first state scale * w q do^T.
    The weight is off by 2^-24, its product with a value by 2^-24, two fp16 terms leave 2^-22, two exact products are added (2^-22 where bits are
    cut off), and scale and its product are off by 2^-24 each: 0.82 * 2^-20 of S.  Where other rows of a column have larger weighted values,
    fp16's smallest numbers leave 2^-50 of the largest of them besides."""
    for row in (0, n - 2, n - 1):
        for others in (False, True):
            thick = one_row(dim, n, row, size, others, row)                  # values, or gradients of outputs
            thin = one_row(dim, n, row, 0.5, not others, row + 1)            # keys, or queries
            g = torch.tensor([decay], device="cuda")
            behind = torch.arange(1, n + 1, device="cuda") if back else torch.arange(n - 1, -1, -1, device="cuda")
            w = torch.exp(g.double() * behind)[:, None]
            rest = torch.zeros(1, 1, n, dim, dtype=torch.float16, device="cuda")
            got = torch.full((1, 1, dim, dim), math.nan, device="cuda")
            if back:
                outs = [torch.empty_like(rest) for _ in range(3)]
                backend.LinearAttentionBackward(GpuBuffer(thick), GpuBuffer(thin), GpuBuffer(rest), GpuBuffer(rest.clone()), *(GpuBuffer(x) for x in outs),
                                                GpuBuffer(g), 1, 1, 1, n, dim, dim, gradInitialStates=GpuBuffer(got))
                w = w * dim ** -0.5
            else:
                backend.LinearAttention(GpuBuffer(rest), GpuBuffer(thin), GpuBuffer(thick), GpuBuffer(torch.empty_like(rest)), GpuBuffer(g), 1, 1, 1, n, dim,
                                        dim, finalStates=GpuBuffer(got))
            a, b = thin[0, 0].double(), thick[0, 0].double() * w
            ref = a[row][:, None] * b[row][None, :]
            floor = a[row].abs()[:, None] * b.abs().amax(0)[None, :] * 2.0 ** -50 if others else 0.0
            off = (got[0, 0].double() - ref).abs()
            assert bool((off <= 2.0 ** -20 * ref.abs() + floor).all()), (row, others, float((off / ref.abs()).nan_to_num().max()))


@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_fp16_values_stay_in_their_columns(backend, dim):
    """A column's own scale: an infinity or NaN in one column of the values leaves the states' other columns as they were."""
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = ((torch.randn((1, 2, 150, dim), generator=g, device="cuda") * 0.5).half() for _ in range(3))
    decay, out = torch.tensor([-0.01, -0.3], device="cuda"), torch.empty_like(q)

    def states():
        last = torch.empty(1, 2, dim, dim, device="cuda")
        backend.LinearAttention(*(GpuBuffer(x) for x in (q, k, v, out, decay)), 1, 2, 2, 150, dim, dim, finalStates=GpuBuffer(last))
        return last

    clean = states()
    for bad in (math.inf, math.nan):
        v[0, 1, 70, 5] = bad
        last = states()
        hit = torch.zeros_like(last, dtype=torch.bool)
        hit[0, 1, :, 5] = True
        assert torch.equal(last[~hit], clean[~hit]) and not bool(torch.isfinite(last[hit]).any())


# ---- waits that ran out, and several streams -------------------------------------------------------------------------

def test_every_stream_is_told_of_a_wait_that_ran_out():
    """A call on one stream gives up: a poll of another stream tells that stream, and takes the report from neither the first one nor a third."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    backends = [CudaBackend(stream=s) for s in streams]
    x = [[(torch.randn(1, 2, 100, 64, device="cuda") * 0.5).bfloat16() for _ in range(4)] for _ in streams]
    torch.cuda.synchronize()

    def call(i):
        backends[i].LinearAttention(*(GpuBuffer(t) for t in x[i]), None, 1, 2, 2, 100, 64, 64)

    def told(i):
        try:
            backends[i].LinearAttentionPoll()
        except N.AidnError as e:
            assert e.status == N.ETIMEOUT
            return True
        return False

    for i in range(3):
        call(i)
        told(i)   # (of what tests before this one may have left to tell)
    assert not any(told(i) for i in range(3))
    assert N.load().aidn_sdpa_debug_set(None, None, 5) == N.OK
    call(0)
    call(1)
    streams[0].synchronize()
    assert told(1) and told(0) and told(2)
    assert not any(told(i) for i in range(3))
    right = x[1][3].clone()
    call(0)
    call(1)
    assert not told(0) and not told(1)
    assert torch.equal(x[1][3], right)
    try:
        N.linear_attention_poll(torch.cuda.current_stream().cuda_stream)   # (the stream of other tests is told here, not there)
    except N.AidnError:
        pass


def test_a_poll_within_a_capture_leaves_it(backend):
    """A stream that is being captured cannot be waited for: the poll says so, and the capture goes on."""
    stream = torch.cuda.Stream()
    own = CudaBackend(stream=stream)
    x = [(torch.randn(1, 2, 100, 64, device="cuda") * 0.5).bfloat16() for _ in range(4)]
    torch.cuda.synchronize()
    call = lambda: own.LinearAttention(*(GpuBuffer(t) for t in x), None, 1, 2, 2, 100, 64, 64)  # noqa: E731
    call()
    torch.cuda.synchronize()
    right = x[3].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
        with pytest.raises(N.AidnError) as e:
            own.LinearAttentionPoll()
    assert e.value.status == N.EINVAL
    x[3].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x[3], right)
    del graph


_CHECKED = """
import torch
from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
b, other = CudaBackend(), CudaBackend(stream=torch.cuda.Stream())
x = [(torch.randn(1, 2, 100, 64, device="cuda") * 0.5).bfloat16() for _ in range(4)]
torch.cuda.synchronize()
go = lambda b: b.LinearAttention(*(GpuBuffer(t) for t in x), None, 1, 2, 2, 100, 64, 64)
go(b); go(other)
assert N.load().aidn_sdpa_debug_set(None, None, 5) == N.OK
try:
    go(b)
    raise SystemExit("the call did not report the wait that ran out")
except N.AidnError as e:
    assert e.status == N.ETIMEOUT and "LAUNCH-FAULT" in e.message, (e.status, e.message)
go(b); b.LinearAttentionPoll()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=other.stream):
    go(other)
graph.replay(); torch.cuda.synchronize()
print("launch check ok")
"""


def test_launch_check_reports_a_wait_that_ran_out():
    """With AIDOTNET_KERNEL_LAUNCH_CHECK the call itself reports it, once; calls that are captured are not checked.  (The variable is read once.)"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, AIDOTNET_KERNEL_LAUNCH_CHECK="1", PYTHONPATH=root)
    r = subprocess.run([sys.executable, "-c", _CHECKED], capture_output=True, text=True, timeout=300, env=env, cwd=root)
    assert r.returncode == 0 and "launch check ok" in r.stdout, f"stdout:\n{r.stdout}\nstderr:\n{r.stderr[-2000:]}"


# ---- rotary positions far out ----------------------------------------------------------------------------------------

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


@pytest.mark.parametrize("base", [10000.0, 2.0])
def test_far_positions_are_as_exact_as_near_ones(backend, base):
    """Angles reduced in whole numbers: test_gpu_rotary's bound, 2^-21 of the pair's magnitudes, at every position that 64 bits hold."""
    pos = [0, 1, 12345, (1 << 31) - 1, 1 << 31, (1 << 40) + 12345, -(1 << 40) - 7, (1 << 47) + 1, (1 << 52) + 3, (1 << 53) - 1, -(1 << 53) + 1]
    f = backend.RotaryFrequencies(64, base)
    left = [[Fraction(w) * p % TWO_PI for w in f.tensor.tolist()] for p in pos]
    c, s = (torch.tensor([[fn(float(a)) for a in row] for row in left], dtype=torch.float64, device="cuda")[:, None] for fn in (math.cos, math.sin))
    x = torch.randn(len(pos), 3, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y = torch.empty_like(x)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(y), None, None, f, len(pos), 3, 0, 64, positions=GpuBuffer(torch.tensor(pos, device="cuda")))
    a, b = x.double()[..., ::2], x.double()[..., 1::2]
    for got, ref in ((y[..., ::2], a * c - b * s), (y[..., 1::2], a * s + b * c)):
        assert bool(((got.double() - ref).abs() <= 2.0 ** -24 * ref.abs() + 2.0 ** -21 * (a.abs() + b.abs())).all())


# ---- packed rows whose seq_len is a bound ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,key,value,heads", [("bf16", 64, 64, 4), ("f16", 128, 64, 2), ("f32", 40, 72, 4)])
def test_a_bound_on_packed_sequences_changes_nothing(backend, dtype, key, value, heads):
    """seq_len as large as it may be, against seq_len as long as there are rows: the same plan, and so the same bits; and no workspace for rows that are not there."""
    g = torch.Generator(device="cuda").manual_seed(7)
    n, lens = 260, [0, 3, 200, 57]
    q, k, v, do = ((torch.randn((n, h, d), generator=g, device="cuda") * 0.5).to(TORCH_DT[dtype]) for h, d in ((heads, key), (1, key), (1, value), (heads, value)))
    starts = torch.tensor([sum(lens[:i]) for i in range(5)], dtype=torch.int32, device="cuda")
    decay, got = torch.linspace(-0.2, -0.01, heads, device="cuda"), []
    for seq in (n, 0x7fffffff):
        block = N.linear_block(batch=4, heads=heads, kv_heads=1, seq_len=seq, key_dim=key, value_dim=value, dtype=N.BF16 if dtype == "bf16" else N.F16
                               if dtype == "f16" else N.F32, token_starts=starts.data_ptr(), tokens=n)
        outs = [torch.zeros_like(x) for x in (do, q, k, v)]
        last = torch.zeros(4, heads, key, value, device="cuda")
        ins, at = [GpuBuffer(x) for x in (q, k, v)], [GpuBuffer(x) for x in outs]
        backend.LinearAttention(*ins, at[0], GpuBuffer(decay), 4, heads, 1, seq, key, value, tokenStarts=GpuBuffer(starts), finalStates=GpuBuffer(last))
        backend.LinearAttentionBackward(GpuBuffer(do), *ins, *at[1:], GpuBuffer(decay), 4, heads, 1, seq, key, value, tokenStarts=GpuBuffer(starts))
        got.append((N.linear_workspace_bytes(block), N.linear_workspace_bytes(N.linear_bwd_block(block)), *outs, last))
    assert got[0][:2] == got[1][:2]
    for a, b in zip(got[0][2:], got[1][2:]):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("part", [128, 32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("seed", [0, 1])
def test_fp16_results_below_its_normal_numbers(backend, part, interleaved, seed):
    """Rows of a packed projection.  test_gpu_rotary's bound, and fp16's own: below 2^-14 its numbers are 2^-24 apart, and a rounding is off by 2^-25."""
    x = torch.randn(19, 12, 128, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    x = (x * 2.0 ** -torch.arange(19, device="cuda")[:, None, None]).half()   # rows of ever smaller values
    out, f = torch.empty(19, 10, 128, dtype=x.dtype, device="cuda"), backend.RotaryFrequencies(part)
    backend.RotaryEmbedding(GpuBuffer(x), GpuBuffer(out), None, None, f, 19, 10, 0, 128, interleaved=interleaved, queryStride=(12 * 128, 128))
    y, angle = x[:, :10].double(), torch.arange(19, device="cuda").double()[:, None] * f.tensor
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    at, bt = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = y[..., at], y[..., bt]
    for got, ref in ((out[..., at], a * c - b * s), (out[..., bt], a * s + b * c)):
        most = (2.0 ** -11 * ref.abs()).clamp(min=2.0 ** -25) + 2.0 ** -21 * (a.abs() + b.abs())
        assert bool(((got.double() - ref).abs() <= most).all())
    assert torch.equal(out[..., part:], x[:, :10, part:])


# ---- what a backend counts and passes on -----------------------------------------------------------------------------

def prompt(backend, dtype, n, heads, kv, key, value, backward=False):
    """A prompt of one sequence, or its gradients; kernels by the backend's count."""
    make = lambda h, d: GpuBuffer((torch.randn(1, h, n, d, device="cuda") * 0.5).to(TORCH_DT[dtype]))  # noqa: E731
    q, k, v, o = make(heads, key), make(kv, key), make(kv, value), make(heads, value)
    before = backend.launch_count
    if backward:
        backend.LinearAttentionBackward(o, q, k, v, make(heads, key), make(kv, key), make(kv, value), None, 1, heads, kv, n, key, value)
    else:
        backend.LinearAttention(q, k, v, o, None, 1, heads, kv, n, key, value)
    return backend.launch_count - before


@pytest.mark.parametrize("args,forward,backward", [
    (("bf16", 100, 4, 4, 64, 64), 1, 1),      # the scans
    (("bf16", 100, 4, 2, 64, 64), 1, 2),      # and the sums of shared heads
    (("bf16", 100, 4, 2, 64, 128), 1, 3),     # scans of two sizes are two launches
    (("bf16", 4096, 1, 1, 128, 128), 3, 3),   # in segments: what each adds, the states before them, the scans
    (("f32", 4096, 2, 1, 40, 72), 3, 4),
    (("f32", 20, 2, 2, 40, 72), 1, 1)])
def test_launch_count_is_what_ran(backend, args, forward, backward):
    assert prompt(backend, *args) == forward
    assert prompt(backend, *args, backward=True) == backward


@pytest.mark.parametrize("path", [N.PATH_AUTO, N.PATH_GENERIC, N.PATH_DECODE, N.PATH_PREFILL_SM100])
def test_a_forced_attention_path_is_no_path_of_linear_attention(path):
    """A backend may be held to one kernel of softmax attention; linear attention has two paths, and heeds GENERIC."""
    own = CudaBackend(path=path)
    q, k, v = ((torch.randn(1, 2, 90, 64, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda") * 0.5).bfloat16() for i in range(3))
    outs = []
    for b in (own, CudaBackend(path=N.PATH_GENERIC if path == N.PATH_GENERIC else N.PATH_AUTO)):
        out, grads = torch.empty_like(q), [torch.empty_like(q) for _ in range(3)]
        b.LinearAttention(*(GpuBuffer(x) for x in (q, k, v, out)), None, 1, 2, 2, 90, 64, 64)
        b.LinearAttentionBackward(*(GpuBuffer(x) for x in (out, q, k, v, *grads)), None, 1, 2, 2, 90, 64, 64)
        outs.append((out, *grads))
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(*outs))


_THREADS = """
import threading
import torch
from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
backends = [CudaBackend(stream=torch.cuda.Stream()) for _ in range(16)]
x = [[(torch.randn(3, 2, 64, device="cuda") * 0.5).bfloat16() for _ in range(4)] for _ in backends]
states = [torch.zeros(3, 2, 64, 64, device="cuda") for _ in backends]
torch.cuda.synchronize()
gate, failed = threading.Barrier(len(backends)), []

def first(i):
    gate.wait()
    try:
        backends[i].LinearAttentionStep(*(GpuBuffer(t) for t in x[i]), GpuBuffer(states[i]), None, 3, 2, 2, 64, 64)
    except Exception as e:
        failed.append(e)

threads = [threading.Thread(target=first, args=(i,)) for i in range(len(backends))]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not failed, failed
for (q, k, v, out), s in zip(x, states):
    assert torch.equal(s, k.float()[..., None] * v.float()[..., None, :])
print("threads ok")
"""


def test_first_calls_of_many_threads():
    """Calls without a handle learn what the device is when the first of them runs: sixteen first calls at once, in a process of their own."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _THREADS], capture_output=True, text=True, timeout=300, env=dict(os.environ, PYTHONPATH=root), cwd=root)
    assert r.returncode == 0 and "threads ok" in r.stdout, f"stdout:\n{r.stdout}\nstderr:\n{r.stderr[-2000:]}"


# ---- packed rows in buffers with room to spare -----------------------------------------------------------------------

def test_packed_rows_in_larger_buffers(backend):
    """A query buffer kept for more rows than this batch has, beside keys and values that are just large enough."""
    n, lens, starts = 90, (40, 50), torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
    make = lambda rows, h: (torch.randn(rows, h, 64, generator=torch.Generator(device="cuda").manual_seed(rows + h), device="cuda") * 0.5).bfloat16()  # noqa: E731
    q, k, v, do = make(128, 4), make(n, 2), make(n, 2) + 1, make(128, 4) - 1
    sizes = (2, 4, 2, max(lens), 64, 64)
    got = []
    for roomy in (True, False):
        qq, dd = (q, do) if roomy else (q[:n].contiguous(), do[:n].contiguous())
        out, grads = torch.full_like(qq, 7.0), [torch.full_like(x, 7.0) for x in (qq, k, v)]
        kw = dict(tokenStarts=GpuBuffer(starts), **(dict(tokens=n) if roomy else {}))
        backend.LinearAttention(*(GpuBuffer(x) for x in (qq, k, v, out)), None, *sizes, **kw)
        backend.LinearAttentionBackward(*(GpuBuffer(x) for x in (dd, qq, k, v, *grads)), None, *sizes, **kw)
        assert all(bool((x[n:] == 7.0).all()) for x in (out, *grads))
        got.append([x[:n] for x in (out, *grads)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    bufs = [GpuBuffer(x) for x in (q, k, v, torch.empty_like(q))]
    for change in (dict(tokens=91, tokenStarts=GpuBuffer(starts)), dict(tokens=-1, tokenStarts=GpuBuffer(starts)), dict(tokens=5), dict(tokenStarts=GpuBuffer(starts))):
        with pytest.raises(ValueError, match="tokens must be|key is smaller"):
            backend.LinearAttention(*bufs, None, *sizes, **change)
    for change in (dict(tokens=91, tokenStarts=GpuBuffer(starts)), dict(tokens=5)):
        with pytest.raises(ValueError, match="tokens must be|key is smaller"):
            backend.LinearAttentionBackward(GpuBuffer(do), *bufs[:3], *(GpuBuffer(torch.empty_like(x)) for x in (q, k, v)), None, *sizes, **change)


# ---- devices ---------------------------------------------------------------------------------------------------------

class Elsewhere:
    """A buffer that says it is on another device (there is one here)."""

    def __init__(self, tensor):
        self.real = tensor

    @property
    def tensor(self):
        return self

    def get_device(self):
        return 1

    def __getattr__(self, name):
        return getattr(self.real, name)


def calls_by_name(backend):
    """Each method with arguments that are right: (method, its buffers, what else it takes)."""
    x = lambda *s: GpuBuffer(torch.zeros(s, device="cuda"))  # noqa: E731
    ints = lambda *v: GpuBuffer(torch.tensor(v, dtype=torch.int32, device="cuda"))  # noqa: E731
    sizes = dict(batch=1, heads=2, kvHeads=2, keyDim=64, valueDim=64)
    rotary = dict(tokens=4, heads=2, kvHeads=2, headDim=64)
    f = backend.RotaryFrequencies(64)
    return [
        (backend.RotaryEmbedding, dict(query=x(4, 2, 64), queryOut=x(4, 2, 64), key=x(4, 2, 64), keyOut=x(4, 2, 64), frequencies=f, positions=ints(0, 1, 2, 3)), rotary),
        (backend.RotaryEmbeddingBackward, dict(gradQueryOut=x(4, 2, 64), gradQuery=x(4, 2, 64), gradKeyOut=x(4, 2, 64), gradKey=x(4, 2, 64), frequencies=f), rotary),
        (backend.LinearAttention, dict(query=x(1, 2, 8, 64), key=x(1, 2, 8, 64), value=x(1, 2, 8, 64), output=x(1, 2, 8, 64), decay=x(2), lengths=ints(8),
                                       initialStates=x(1, 2, 64, 64), finalStates=x(1, 2, 64, 64), stateSlots=ints(0)), dict(seqLen=8, **sizes)),
        (backend.LinearAttention, dict(query=x(8, 2, 64), key=x(8, 2, 64), value=x(8, 2, 64), output=x(8, 2, 64), decay=x(2), tokenStarts=ints(0, 8)),
         dict(seqLen=8, **sizes)),
        (backend.LinearAttentionBackward, dict(gradOutput=x(1, 2, 8, 64), query=x(1, 2, 8, 64), key=x(1, 2, 8, 64), value=x(1, 2, 8, 64), gradQuery=x(1, 2, 8, 64),
                                               gradKey=x(1, 2, 8, 64), gradValue=x(1, 2, 8, 64), decay=x(2), initialStates=x(1, 2, 64, 64),
                                               gradFinalStates=x(1, 2, 64, 64), gradInitialStates=x(1, 2, 64, 64)), dict(seqLen=8, **sizes)),
        (backend.LinearAttentionStep, dict(query=x(1, 2, 64), key=x(1, 2, 64), value=x(1, 2, 64), output=x(1, 2, 64), states=x(1, 2, 64, 64), decay=x(2),
                                           stateSlots=ints(0)), sizes)]


def test_buffers_of_another_device_are_refused(backend):
    for method, buffers, rest in calls_by_name(backend):
        method(**buffers, **rest)
        for name, buf in buffers.items():
            with pytest.raises(ValueError, match="device"):
                method(**{**buffers, name: Elsewhere(buf.tensor)}, **rest)


def test_another_device_may_be_the_current_one(backend, monkeypatch):
    """Calls without a handle run on the current device: a backend makes its own the current one for them, where it is not."""
    entered, current = [], [0]

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            current[0] = self.device

        def __exit__(self, *_):
            current[0] = 1

    calls = calls_by_name(backend)
    for method, buffers, rest in calls:
        method(**buffers, **rest)
    backend.LinearAttentionPoll()
    stream = torch.cuda.current_stream()   # (before the current device is another)
    own = CudaBackend(stream=stream)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    current[0] = 1
    for method, buffers, rest in calls:
        entered.clear()
        getattr(own, method.__name__)(**buffers, **rest)
        assert entered and set(entered) == {0}, method.__name__
    entered.clear()
    own.LinearAttentionPoll()
    assert entered == [0]


# ---- refusals, one thing changed in each -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float64, torch.int16])
def test_types_that_are_not_served(backend, dtype):
    for method, buffers, rest in calls_by_name(backend):
        small = ("decay", "frequencies", "positions", "lengths", "tokenStarts", "stateSlots")
        other = {n: b if n in small or "tates" in n else GpuBuffer(b.tensor.to(dtype)) for n, b in buffers.items()}
        with pytest.raises(ValueError, match="not served"):
            method(**other, **rest)


def test_buffers_that_are_too_small_by_name(backend):
    """Each buffer one element short, everything else right: the error names it."""
    names = dict(queryOut="query", keyOut="key", gradQueryOut="query", gradQuery="query", gradKeyOut="key", gradKey="key")   # (a rotation names the pair)
    for method, buffers, rest in calls_by_name(backend):
        rotary = "Rotary" in method.__name__
        for name, buf in buffers.items():
            if name == "frequencies":
                continue   # (fewer of them turn a smaller part)
            if name == "query" and "tokenStarts" in buffers:
                continue   # (it says how many rows there are)
            short = GpuBuffer(buf.tensor.reshape(-1)[:-1].clone())
            step = method.__name__ == "LinearAttentionStep" and name in ("query", "key", "value", "output")
            match = "smaller" if step else names.get(name, name) if rotary else name
            with pytest.raises(ValueError, match=match):
                method(**{**buffers, name: short}, **rest)


def test_types_of_decay_and_gradients_by_name(backend):
    for method, buffers, rest in calls_by_name(backend):
        for name in ("decay", "gradKey", "gradQuery", "gradValue", "initialStates", "finalStates", "gradFinalStates", "gradInitialStates", "states"):
            if name in buffers and "Rotary" not in method.__name__:
                with pytest.raises(ValueError, match=name):
                    method(**{**buffers, name: GpuBuffer(buffers[name].tensor.half())}, **rest)


# ---- slices of 64 columns that are not full --------------------------------------------------------------------------

# (On 148 SMs slices of 64 columns are taken here, one wave of CTAs against two of slices of 32; the last slice has 8, 32 or 40 columns.  Uncut: there are CTAs
# enough.  heads is for the forward pass; a gradient's three scans reach the same with a third of them.)
WIDE = [(136, 136, 96, 32), (256, 96, 64, 32), (256, 40, 100, 34)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("key,value,items,_", WIDE)
def test_slices_that_are_not_full(backend, dtype, key, value, items, _):
    check_forward(backend, Case(dtype, [70, 33], items // 2, items // 2, key, value, "starts", first=True, seed=30))
    check_forward(backend, Case(dtype, [40, 64], items // 2, 1, key, value, "lengths_token", first=True, seed=31))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("key,value,_,items", WIDE)
def test_slices_that_are_not_full_backward(backend, dtype, key, value, _, items):
    check_backward(backend, Case(dtype, [70, 33], items // 2, items // 2, key, value, "starts", first=True, seed=32), last=True)


# ---- lengths and starts that are none --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f16", 128), ("f32", 40)])
def test_lengths_beyond_the_ends_are_taken_to_them(backend, dtype, dim):
    """A length below 0 is 0, one above seq_len is seq_len; starts before the first row or behind the last are those rows.  Nothing outside is written."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = [(torch.randn((3, 2, 70, dim), generator=g, device="cuda") * 0.5).to(TORCH_DT[dtype]) for _ in range(3)]
    ints = lambda *v: GpuBuffer(torch.tensor(v, dtype=torch.int32, device="cuda"))  # noqa: E731
    big = (1 << 31) - 1
    for kw in ((dict(lengths=ints(-3, 1000, 33)), dict(lengths=ints(0, 70, 33))), (dict(lengths=ints(-big, big, 1)), dict(lengths=ints(0, 70, 1))),
               (dict(tokenStarts=ints(-5, 30, 40, 5000)), dict(tokenStarts=ints(0, 30, 40, 210)))):
        got = []
        for k in kw:
            seq = 70 if "lengths" in k else 210
            made = [guarded(x[0].shape, x[0].dtype, "cuda", 3.0) for _ in range(4)]
            bufs = [GpuBuffer(t) for t in x]
            backend.LinearAttention(*bufs, GpuBuffer(made[0][1]), None, 3, 2, 2, seq, dim, dim, **k)
            backend.LinearAttentionBackward(bufs[0], *bufs, *(GpuBuffer(m[1]) for m in made[1:]), None, 3, 2, 2, seq, dim, dim, **k)
            for flat, _ in made:
                check_guards(flat, "out or gradient")
            got.append([m[1] for m in made])
        assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(*got))


# ---- graphs that share a stream and a backend ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 40)])
def test_two_graphs_replayed_at_once(dtype, dim):
    """Two graphs recorded one after the other on one stream by one backend, with workspaces for segments and for shared heads, replayed on two streams at
    once, beside eager calls of the same backend: all as alone."""
    stream = torch.cuda.Stream()
    own, plain = CudaBackend(stream=stream), CudaBackend()
    g = torch.Generator(device="cuda").manual_seed(11)
    sets = []
    for n in (2500, 1700, 2100):
        ins = [(torch.randn((1, h, n, dim), generator=g, device="cuda") * 0.3).to(TORCH_DT[dtype]) for h in (2, 1, 1, 2)]
        sets.append((n, ins, [torch.zeros_like(t) for t in (ins[0], ins[0], ins[1], ins[2])]))

    def calls(backend, which):
        n, (q, k, v, do), (out, *grads) = sets[which]
        backend.LinearAttention(*(GpuBuffer(t) for t in (q, k, v, out)), None, 1, 2, 1, n, dim, dim)
        backend.LinearAttentionBackward(*(GpuBuffer(t) for t in (do, q, k, v, *grads)), None, 1, 2, 1, n, dim, dim)

    right = []
    for i in range(3):
        calls(plain, i)
        right.append([t.clone() for t in sets[i][2]])
    torch.cuda.synchronize()
    calls(own, 2)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=stream):
            calls(own, i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for _, _, outs in sets:
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        calls(own, 2)
        torch.cuda.synchronize()
        for i in range(3):
            assert all(torch.equal(a, b) for a, b in zip(sets[i][2], right[i])), i
    del graphs


# ---- batches that are taken from the longest sequence on -------------------------------------------------------------

@pytest.mark.parametrize("dtype,key,value", [("bf16", 64, 64), ("bf16", 128, 128), ("f16", 64, 128)])
@pytest.mark.parametrize("layout", ["starts", "lengths", "lengths_token"])
@pytest.mark.parametrize("lens", [[3, 0, 200, 64, 200], [70, 71], [0, 0, 0, 1], list(range(1, 65))])
def test_ragged_batches_of_more_sequences_and_heads_than_sms(backend, dtype, key, value, layout, lens):
    """(The order is by lengths here; of equal ones the first is first.)  Every sequence has its rows and its states."""
    heads = 4 if len(lens) == 64 else 100
    check_forward(backend, Case(dtype, lens, heads, heads // 2, key, value, layout, first=True, seed=40))
    check_backward(backend, Case(dtype, lens, heads, heads, key, value, layout, seed=41), last=True)


def test_ragged_batch_by_slots(backend):
    """The same with states by slot: a slot is an earlier sequence's by the batch's order, whatever the order on the device."""
    lens, heads = [20, 90, 150, 7], 60
    c = Case("bf16", lens, heads, heads, 64, 64, "starts", seed=42)
    pool = torch.randn(4, heads, 64, 64, generator=c.g, device="cuda")
    was, out = pool.clone(), torch.empty(c.shape(heads, 64), dtype=torch.bfloat16, device="cuda")
    slots = GpuBuffer(torch.tensor([2, 2, -1, 0], dtype=torch.int32, device="cuda"))
    backend.LinearAttention(c.buf(c.q), c.buf(c.k), c.buf(c.v), GpuBuffer(out), c.buf(c.decay), *c.sizes(), initialStates=GpuBuffer(pool),
                            finalStates=GpuBuffer(pool), stateSlots=slots, **c.kw())
    for b, nan in enumerate((False, True, False, False)):
        assert bool((torch.isnan if nan else torch.isfinite)(c.of(out, b)).all()), b
    assert torch.equal(pool[[1, 3]], was[[1, 3]]) and not torch.equal(pool[0], was[0]) and not torch.equal(pool[2], was[2])


# ---- a layer from a packed projection --------------------------------------------------------------------------------

def test_a_layer_from_a_packed_projection(backend):
    """Prompts of unequal lengths and the tokens that follow them: rotation out of the packed rows, values copied, states by slot, single tokens from there.  The
    rotated rows are held against the formula, and what is computed of them against the recurrence of whole sequences."""
    heads, kvHeads, headDim, lens, extra = 4, 2, 64, [70, 3, 130], 3
    batch, tokens, longest = len(lens), sum(lens), max(lens)
    g = torch.Generator(device="cuda").manual_seed(50)
    project = lambda n: (torch.randn((n, heads + 2 * kvHeads, headDim), generator=g, device="cuda") * 0.5).bfloat16()  # noqa: E731
    dense = lambda n, h: GpuBuffer(torch.empty(n, h, headDim, dtype=torch.bfloat16, device="cuda"))  # noqa: E731
    ints = lambda x: GpuBuffer(torch.tensor(x, dtype=torch.int32, device="cuda"))  # noqa: E731
    begin = [sum(lens[:i]) for i in range(batch + 1)]
    decay, starts, slots = GpuBuffer(torch.tensor([-0.3, -0.1, -0.02, -0.001], device="cuda")), ints(begin), ints([4, 0, 2])
    pool = GpuBuffer(torch.zeros(6, heads, headDim, headDim, device="cuda"))
    f = backend.RotaryFrequencies(rotaryDim=64, scaling="parts", factor=8.0, originalLength=4096)
    row = ((heads + 2 * kvHeads) * headDim, headDim)

    def split(qkv, q, k, tokens, positions):
        flat = qkv.view(-1)
        backend.RotaryEmbedding(GpuBuffer(flat), q, GpuBuffer(flat[heads * headDim:]), k, f, tokens, heads, kvHeads, headDim, positions=positions,
                                queryStride=row, keyStride=row)
        for got, ins in ((q, qkv[:, :heads]), (k, qkv[:, heads:heads + kvHeads])):
            check_turned(got.tensor, *formula(ins, f.tensor, positions.tensor, True, 1.0), "bf16")
        return GpuBuffer(qkv[:, heads + kvHeads:].contiguous())

    q, k, out = dense(tokens, heads), dense(tokens, kvHeads), dense(tokens, heads)
    v = split(project(tokens), q, k, tokens, ints([t for n in lens for t in range(n)]))
    backend.LinearAttention(q, k, v, out, decay, batch, heads, kvHeads, longest, headDim, headDim, tokenStarts=starts, initialStates=pool,
                            finalStates=pool, stateSlots=slots)
    all_rows = [[x.tensor[begin[b]:begin[b + 1]] for x in (q, k, v, out)] for b in range(batch)]
    for t in range(extra):
        q1, k1, out1 = dense(batch, heads), dense(batch, kvHeads), dense(batch, heads)
        v1 = split(project(batch), q1, k1, batch, ints([n + t for n in lens]))
        backend.LinearAttentionStep(q1, k1, v1, out1, pool, decay, batch, heads, kvHeads, headDim, headDim, stateSlots=slots)
        for b in range(batch):
            all_rows[b] = [torch.cat((x, y.tensor[b:b + 1])) for x, y in zip(all_rows[b], (q1, k1, v1, out1))]
    for b, n in enumerate(lens):
        qq, kk, vv = (x.double().transpose(0, 1).repeat_interleave(heads // x.shape[1], 0) for x in all_rows[b][:3])
        lam = decay.tensor.double()
        ref, state = recurrence(qq, kk, vv, lam, headDim ** -0.5)
        size, size_s = recurrence(qq.abs(), kk.abs(), vv.abs(), lam, headDim ** -0.5)
        u, e = 2.0 ** -8, e32(headDim, n + extra)
        near(all_rows[b][3].transpose(0, 1), ref, (u + e) * size, u, f"sequence {b}", 3 * u)
        near(pool.tensor[[4, 0, 2][b]], state, (4 * u * u + e) * size_s, 2.0 ** -24, f"state of sequence {b}", 1e-5)
    assert bool((pool.tensor[[1, 3, 5]] == 0).all())


# ---- what is rounded on the way to a 16-bit output -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("key,value", [(64, 64), (128, 128), (64, 128), (128, 64)])
@pytest.mark.parametrize("lens", [[64, 64], [50, 50], [1, 1]])
def test_weighted_products_are_not_rounded(backend, dtype, key, value, lens):
    """Behind no state, an output is a sum of weighted products with values: two terms of the type hold a product to u^2 of itself, so that what is left is fp32's
    errors (test_gpu_linear's e32) and one rounding.  Gradients as well."""
    u, heads = torch.finfo(TORCH_DT[dtype]).eps / 2, 4
    c = Case(dtype, lens, heads, heads, key, value, "head", seed=60)
    out, grads = torch.empty_like(c.do), [torch.empty_like(x) for x in (c.q, c.k, c.v)]
    backend.LinearAttention(*(GpuBuffer(x) for x in (c.q, c.k, c.v, out, c.decay)), *c.sizes())
    backend.LinearAttentionBackward(*(GpuBuffer(x) for x in (c.do, c.q, c.k, c.v, *grads, c.decay)), *c.sizes())
    most = 2 * u * u + e32(max(key, value), lens[0])
    for b in range(2):
        def run(ins, do):
            ins = [x.requires_grad_() for x in ins]
            ref = recurrence(*ins, c.log_decay(), key ** -0.5)[0]
            return (ref.detach(), *torch.autograd.grad((ref * do).sum(), ins))
        wide = [x[b].double() for x in (c.q, c.k, c.v)]
        refs, sizes = run(wide, c.do[b].double()), run([x.abs().detach() for x in wide], c.do[b].double().abs())
        for name, got, ref, size in zip(("out", "dq", "dk", "dv"), (out, *grads), refs, sizes):
            near(got[b], ref, most * size, u, name)


def test_amplitude_of_zero(backend):
    """It would be a factor of 0; the argument block takes 0 for 1."""
    for method, buffers, rest in calls_by_name(backend):
        if "Rotary" in method.__name__:
            with pytest.raises(ValueError, match="amplitude"):
                method(**buffers, **rest, amplitude=0.0)
