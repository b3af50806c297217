"""Rotary positions and linear attention without a GPU: structs against the header, refused arguments, frequencies."""
import math
import os
import subprocess

import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(os.path.join(ROOT, "aidotnet", "tensors_b200", "lib", "libaidotnet_sdpa_sm100.so")):
        pytest.skip("library not built")
    return N.load()


def test_structs_match_the_header(tmp_path):
    """Sizes, and field by field the offsets that the C compiler gives."""
    mirrors = {"aidn_rotary_args": N.RotaryArgs, "aidn_linear_args": N.LinearArgs, "aidn_linear_bwd_args": N.LinearBwdArgs,
               "aidn_linear_step_args": N.LinearStepArgs}
    src = ['#include "aidn_sdpa.h"', "#include <stddef.h>", "#include <stdio.h>", "int main(){"]
    expected = []
    for name, mirror in mirrors.items():
        src.append(f'printf("%zu\\n", sizeof({name}));')
        expected.append(N.ctypes.sizeof(mirror))
        for field, _ in mirror._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            expected.append(getattr(mirror, field).offset)
    (tmp_path / "t.c").write_text("\n".join(src + ["return 0;}"]))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()] == expected


def test_packed_blocks_are_the_structs():
    """The blocks that are packed in one go hold every argument in its field."""
    block = N.linear_block(q=1, k=2, v=3, out=4, decay=5, lengths=6, token_starts=7, initial_state=8, final_state=9, state_slots=10,
                           q_stride=(11, 12, 13), k_stride=(14, 15, 16), v_stride=(17, 18, 19), o_stride=(20, 21, 22), tokens=23,
                           seq_len=24, batch=25, heads=26, kv_heads=27, key_dim=28, value_dim=29, dtype=2, num_slots=31, path=1, scale=0.5,
                           workspace=34, workspace_bytes=35)
    a = N.LinearArgs.from_buffer_copy(block)
    got = [getattr(a, n) for n in ("q", "k", "v", "out", "decay", "lengths", "token_starts", "initial_state", "final_state", "state_slots")]
    got += [x for n in ("q_stride", "k_stride", "v_stride", "o_stride") for x in getattr(a, n)]
    got += [a.tokens, a.seq_len, a.batch, a.heads, a.kv_heads, a.key_dim, a.value_dim]
    assert got == list(range(1, 30))
    assert (a.dtype, a.num_slots, a.path, a.scale, a.workspace, a.workspace_bytes) == (2, 31, 1, 0.5, 34, 35)
    b = N.LinearBwdArgs.from_buffer_copy(N.linear_bwd_block(
        block, dout=1, d_final_state=2, dq=3, dk=4, dv=5, d_initial_state=6, do_stride=(7, 8, 9), dq_stride=(10, 11, 12),
        dk_stride=(13, 14, 15), dv_stride=(16, 17, 18)))
    assert b.fwd.q == 1 and b.fwd.workspace_bytes == 35
    assert [b.dout, b.d_final_state, b.dq, b.dk, b.dv, b.d_initial_state] + [x for n in ("do", "dq", "dk", "dv") for x in getattr(b, n + "_stride")] == list(range(1, 19))


ROTARY = dict(query=4096, query_out=8192, frequencies=4096, tokens=4, heads=2, head_dim=64, rotary_dim=64, dtype=N.BF16, stream=0)


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"),
    (dict(heads=0), "heads"),
    (dict(kv_heads=-1), "heads"),
    (dict(head_dim=60), "multiple of 8"),
    (dict(head_dim=264), "multiple of 8"),
    (dict(rotary_dim=0), "rotary_dim"),
    (dict(rotary_dim=7), "rotary_dim"),
    (dict(rotary_dim=66), "rotary_dim"),
    (dict(dtype=5), "dtype"),
    (dict(layout=N.ROPE_NONE), "layout"),
    (dict(positions=4096, position_bytes=2), "position_bytes"),
    (dict(start_position=-1), "start_position"),
    (dict(seq_len=-1), "seq_len"),
    (dict(amplitude=math.inf), "amplitude"),
    (dict(amplitude=math.nan), "amplitude"),
    (dict(query=0), "null"),
    (dict(frequencies=0), "null"),
    (dict(key=4096, kv_heads=2), "come together"),
    (dict(key=4096, key_out=8192), "come together"),
    (dict(kv_heads=2), "come together"),
    (dict(query=4097), "aligned"),
    (dict(frequencies=4100), "aligned"),
    (dict(positions=4100, position_bytes=8), "aligned"),
    (dict(query_stride=(-64, 64)), "negative"),
    (dict(query_out=4096, query_stride=(256, 64)), "in place"),
])
def test_rotary_refuses(lib, change, word):
    """(The addresses are none: a call that got past its checks would have nothing to launch on here.)"""
    with pytest.raises(N.AidnError) as e:
        N.rotary(**{**ROTARY, **change})
    assert word in str(e.value)


def test_rotary_of_nothing_is_no_launch(lib):
    N.rotary(**{**ROTARY, "tokens": 0, "query": 0, "query_out": 0})


LINEAR = dict(q=4096, k=4096, v=4096, out=8192, batch=2, heads=4, kv_heads=2, seq_len=8, key_dim=64, value_dim=64, dtype=N.BF16)
GRADS = dict(dout=4096, dq=8192, dk=8192, dv=8192)
SIZES = [
    (dict(batch=0), "batch"),
    (dict(batch=65536), "65535"),
    (dict(heads=0), "heads"),
    (dict(kv_heads=3), "divide"),
    (dict(key_dim=60), "multiples of 8"),
    (dict(value_dim=264), "multiples of 8"),
    (dict(dtype=7), "dtype"),
    (dict(path=N.PATH_DECODE), "path"),
    (dict(seq_len=0), "seq_len"),
    (dict(seq_len=1 << 31), "seq_len"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(lengths=4096, token_starts=4096), "exclude"),
    (dict(token_starts=4096, tokens=-1), "tokens"),
    (dict(lengths=4098), "aligned"),
    (dict(decay=4098), "aligned"),
    (dict(q=4097), "aligned"),
    (dict(q=0), "null"),
    (dict(k_stride=(1, -1, 1)), "negative"),
    (dict(initial_state=4100), "16-byte"),
    (dict(workspace=4100), "256-byte"),
]


@pytest.mark.parametrize("change,word", SIZES + [(dict(out=0), "null"), (dict(final_state=4100), "16-byte"),
                                                 (dict(state_slots=4096), "num_slots")])
def test_linear_attention_refuses(lib, change, word):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention(N.linear_block(**{**LINEAR, **change}), 0)
    assert word in str(e.value)


@pytest.mark.parametrize("change,word", SIZES)
def test_linear_attention_backward_refuses(lib, change, word):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_backward(N.linear_bwd_block(N.linear_block(**{**LINEAR, **change}), **GRADS), 0)
    assert word in str(e.value)


@pytest.mark.parametrize("change,grads,word,status", [
    (dict(state_slots=4096, num_slots=4), {}, "state_slots", N.EUNSUPPORTED),
    ({}, dict(dout=0), "null", N.EINVAL),
    ({}, dict(dv=0), "null", N.EINVAL),
    ({}, dict(dq=8193), "aligned", N.EINVAL),
    ({}, dict(d_final_state=4100), "16-byte", N.EINVAL),
    ({}, dict(d_initial_state=4100), "16-byte", N.EINVAL),
    ({}, dict(dk_stride=(1, 1, -1)), "negative", N.EINVAL),
    ({}, {}, "workspace", N.EWORKSPACE),   # shared heads need it
    (dict(workspace=4096, workspace_bytes=16), {}, "workspace", N.EWORKSPACE),
])
def test_linear_attention_backward_refuses_its_own(lib, change, grads, word, status):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_backward(N.linear_bwd_block(N.linear_block(**{**LINEAR, **change}), **{**GRADS, **grads}), 0)
    assert word in str(e.value) and e.value.status == status


def test_workspace_sizes(lib):
    """fp32 sums of dk and dv for every query head where heads are shared; sizes that are refused give no number."""
    need = N.linear_workspace_bytes(N.linear_bwd_block(N.linear_block(**LINEAR)))
    assert need >= 2 * 2 * 8 * 4 * 64 * 4
    assert N.linear_workspace_bytes(N.linear_block(**LINEAR)) >= 0
    for block in (N.linear_block(**{**LINEAR, "heads": 0}), N.linear_bwd_block(N.linear_block(**{**LINEAR, "heads": 0}))):
        with pytest.raises(N.AidnError):
            N.linear_workspace_bytes(block)


STEP = dict(q=4096, k=4096, v=4096, out=8192, states=4096, batch=2, heads=4, kv_heads=2, key_dim=64, value_dim=64, dtype=N.BF16, stream=0)


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "batch"),
    (dict(batch=65536), "65535"),
    (dict(kv_heads=0), "kv_heads"),
    (dict(kv_heads=3), "divide"),
    (dict(key_dim=4), "multiples of 8"),
    (dict(value_dim=300), "multiples of 8"),
    (dict(dtype=-1), "dtype"),
    (dict(scale=-0.5), "scale"),
    (dict(state_slots=4096), "num_slots"),
    (dict(states=0), "null"),
    (dict(out=0), "null"),
    (dict(v=4097), "aligned"),
    (dict(state_slots=4098, num_slots=2), "aligned"),
    (dict(states=4104), "16-byte"),
    (dict(o_stride=(-1, 0)), "negative"),
])
def test_step_refuses(lib, change, word):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_step(**{**STEP, **change})
    assert word in str(e.value)


def test_step_of_nothing_is_no_launch(lib):
    N.linear_attention_step(**{**STEP, "batch": 0, "q": 0, "states": 0})


# ---- frequencies -----------------------------------------------------------------------------------------------------

def test_plain_frequencies():
    got = rotary_frequencies(8, 10000.0)
    assert got.dtype == torch.float64
    assert torch.allclose(got, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)


def test_linear_scaling_divides_all():
    assert torch.equal(rotary_frequencies(16, 5000.0, "linear", 4.0), rotary_frequencies(16, 5000.0) / 4)


def test_raised_base_slows_the_slowest_by_the_factor():
    plain, raised = rotary_frequencies(64), rotary_frequencies(64, scaling="base", factor=8.0)
    assert raised[0] == 1 and abs(float(plain[-1] / raised[-1]) - 8) < 1e-12
    assert bool((raised[1:] < plain[1:]).all())


def test_parts_keep_fast_pairs_and_divide_slow_ones():
    plain, parts = rotary_frequencies(128), rotary_frequencies(128, scaling="parts", factor=8.0, originalLength=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    assert torch.equal(parts[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert bool(between.any()) and bool(((parts < plain) & (parts > plain / 8))[between].all())


@pytest.mark.parametrize("args", [dict(rotaryDim=0), dict(rotaryDim=7), dict(rotaryDim=8, base=0.0), dict(rotaryDim=8, factor=-1.0),
                                  dict(rotaryDim=8, scaling="other"), dict(rotaryDim=2, scaling="base"),
                                  dict(rotaryDim=8, scaling="parts"), dict(rotaryDim=8, scaling="parts", originalLength=10, fastTurns=1.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        rotary_frequencies(**args)


# ---- outputs that overlap --------------------------------------------------------------------------------------------

SPREAD = dict(q=4096, k=8192, v=12288, out=16384, batch=2, heads=4, kv_heads=4, seq_len=8, key_dim=64, value_dim=64, dtype=N.BF16)


@pytest.mark.parametrize("change", [dict(query_out_stride=(128, 0)), dict(query_out_stride=(0, 64)), dict(query_out_stride=(127, 64)),
                                    dict(query_out_stride=(64, 64)), dict(query_out=4096, query_stride=(64, 32), query_out_stride=(64, 32)),
                                    dict(key=16384, kv_heads=2, key_out=8192), dict(key=8192, kv_heads=2, key_out=16384),
                                    dict(key=16384, kv_heads=2, key_out=4096),
                                    dict(key=16384, kv_heads=3, key_out=32768, key_out_stride=(160, 64))])
def test_rotary_refuses_outputs_that_overlap(lib, change):
    """(A token stride that leaves no room for its heads, a head stride below the head's size, one buffer for two outputs.)"""
    with pytest.raises(N.AidnError) as e:
        N.rotary(**{**ROTARY, **change})
    assert "overlap" in str(e.value) and e.value.status == N.EINVAL


@pytest.mark.parametrize("change", [dict(out=4096), dict(out=8192), dict(out=12288), dict(o_stride=(2048, 0, 64)), dict(o_stride=(2048, 512, 63)),
                                    dict(o_stride=(511, 64, 256)), dict(o_stride=(64, 2048, 100)), dict(token_starts=256, tokens=9, o_stride=(0, 64, 192))])
def test_linear_attention_refuses_an_output_that_overlaps(lib, change):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention(N.linear_block(**{**SPREAD, **change}), 0)
    assert "overlap" in str(e.value) and e.value.status == N.EINVAL


@pytest.mark.parametrize("grads", [dict(dq=4096), dict(dk=8192), dict(dv=12288), dict(dv=20480), dict(dk=24576), dict(dv=28672), dict(dq=28672),
                                   dict(dq_stride=(2048, 512, 0)), dict(dk_stride=(2048, 63, 256)), dict(dv_stride=(100, 64, 256))])
def test_linear_attention_backward_refuses_gradients_that_overlap(lib, grads):
    made = {**dict(dout=20480, dq=24576, dk=28672, dv=32768), **grads}
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_backward(N.linear_bwd_block(N.linear_block(**SPREAD), **made), 0)
    assert "overlap" in str(e.value) and e.value.status == N.EINVAL


@pytest.mark.parametrize("change", [dict(out=4096), dict(o_stride=(255, 64)), dict(o_stride=(256, 60)), dict(o_stride=(64, 64))])
def test_step_refuses_an_output_that_overlaps(lib, change):
    with pytest.raises(N.AidnError) as e:
        N.linear_attention_step(**{**STEP, **change})
    assert "overlap" in str(e.value) and e.value.status == N.EINVAL


def test_outputs_of_every_order_are_taken(lib):
    """Strides in any order, and any distance where there is one row: what is left to refuse is that there is no device here (or nothing at all)."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are none")
    for stride in ((2048, 512, 64), (2048, 64, 256), (64, 1024, 128), (0, 0, 0)):
        with pytest.raises(N.AidnError) as e:
            N.linear_attention(N.linear_block(**{**SPREAD, "o_stride": stride}), 0)
        assert "overlap" not in str(e.value)
    with pytest.raises(N.AidnError) as e:
        N.linear_attention(N.linear_block(**{**SPREAD, "batch": 1, "seq_len": 1, "o_stride": (1, 64, 1)}), 0)
    assert "overlap" not in str(e.value)


# ---- sizes at the ends -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("change", [dict(seq_len=0x7fffffff), dict(seq_len=0x7fffffc1), dict(token_starts=4096, seq_len=0x7fffffff, tokens=0x7fffffff)])
def test_sequences_that_are_too_long_for_a_count_of_rows(lib, change):
    """What counts a segment's rows has 31 bits, whole chunks of them: a longer sequence would lose its last rows."""
    small = dict(key_dim=8, value_dim=8, heads=1, kv_heads=1, batch=1)
    for call in (lambda b: N.linear_attention(b, 0), N.linear_workspace_bytes):
        with pytest.raises(N.AidnError) as e:
            call(N.linear_block(**{**LINEAR, **small, **change}))
        assert "rows" in str(e.value) and e.value.status == N.EINVAL


def test_workspace_of_sizes_beyond_64_bits(lib):
    """Bytes that 64 bits do not hold are refused, not wrapped around."""
    huge = dict(batch=65535, heads=65535, kv_heads=1, seq_len=0x7fffffc0, key_dim=256, value_dim=256)
    with pytest.raises(N.AidnError) as e:
        N.linear_workspace_bytes(N.linear_bwd_block(N.linear_block(**{**LINEAR, **huge})))
    assert "2^60" in str(e.value)
    block = N.linear_bwd_block(N.linear_block(**{**LINEAR, **dict(batch=1, heads=64, kv_heads=1, seq_len=1 << 20, key_dim=256, value_dim=128)}))
    assert N.linear_workspace_bytes(block) >= (64 << 20) * (256 + 128) * 4
