"""The 8-bit paged cache without a GPU: structs against the header, arguments that are refused before anything is launched."""
import os
import subprocess
import weakref

import pytest
import torch

from aidotnet.tensors_b200 import native as N
from aidotnet.tensors_b200.backend import KvCacheFp8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(os.path.join(ROOT, "aidotnet", "tensors_b200", "lib", "libaidotnet_sdpa_sm100.so")):
        pytest.skip("library not built")
    return N.load()


def test_structs_match_the_header(tmp_path):
    """Sizes, and field by field the offsets that the C compiler gives."""
    mirrors = {"aidn_kv8_cache": N.Kv8Cache, "aidn_kv8_append_args": N.Kv8AppendArgs}
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


def test_rotations_match_the_header(tmp_path):
    (tmp_path / "t.c").write_text('#include "aidn_sdpa.h"\n#include <stdio.h>\n'
                                  'int main(){printf("%d %d %d", AIDN_ROPE_NONE, AIDN_ROPE_INTERLEAVED, AIDN_ROPE_HALVES);return 0;}\n')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()] == [N.ROPE_NONE, N.ROPE_INTERLEAVED, N.ROPE_HALVES]


GOOD = dict(key_pool=4096, value_pool=4096, key_scale=4096, value_scale=4096, block_table=4096, block_table_stride=4, num_blocks=8,
            block_size=16, kv_heads=2, head_dim=64)
ARGS = dict(key=4096, value=4096, start=4096, tokens=2, batch=2, heads=0, dtype=N.BF16, rope=N.ROPE_NONE)


@pytest.mark.parametrize("cache,args,word", [
    (dict(key_pool=0), {}, "null"),
    (dict(value_scale=0), {}, "null"),
    (dict(block_table=0), {}, "null"),
    (dict(block_size=0), {}, "block_size"),
    (dict(block_size=65537), {}, "block_size"),
    (dict(block_table_stride=0), {}, "block_table_stride"),
    (dict(num_blocks=-1), {}, "num_blocks"),
    (dict(kv_heads=0), {}, "kv_heads"),
    (dict(head_dim=0), {}, "head_dim"),
    (dict(head_dim=264), {}, "head_dim"),
    (dict(head_dim=60), {}, "multiple of 8"),
    (dict(pool_stride=(2048, 126, 64)), {}, "strides"),
    (dict(pool_stride=(2048, -128, 64)), {}, "strides"),
    (dict(key_pool=4097), {}, "aligned"),
    ({}, dict(tokens=-1), "tokens"),
    ({}, dict(batch=0), "batch"),
    ({}, dict(tokens=3), "same number"),
    ({}, dict(tokens=1 << 31), "tokens"),
    ({}, dict(dtype=7), "dtype"),
    ({}, dict(rope=3), "rotation"),
    ({}, dict(key=0), "null"),
    ({}, dict(start=0), "null"),
    ({}, dict(query=4096, heads=4), "query_out"),
    ({}, dict(query=4096, query_out=4096), "heads"),
    ({}, dict(rope=N.ROPE_HALVES), "cosine"),
    ({}, dict(key=4097), "aligned"),
    ({}, dict(key_stride=(-64, 64)), "stride"),
])
def test_append_refuses(lib, cache, args, word):
    """(The addresses are none: a call that got past its checks would have nothing to launch on here.)"""
    with pytest.raises(N.AidnError) as e:
        N.kv8_append(N.kv8_cache(**{**GOOD, **cache}), stream=0, **{**ARGS, **args})
    assert word in str(e.value)


def test_append_of_nothing_is_no_launch(lib):
    N.kv8_append(N.kv8_cache(**GOOD), stream=0, **{**ARGS, "tokens": 0, "key": 0, "value": 0, "start": 0})


def test_blocks_of_more_than_2_to_the_31_rows(lib):
    """The strides of a dense pool are 64-bit whatever its block size and heads are: such a pool is taken."""
    N.kv8_append(N.kv8_cache(**{**GOOD, "block_size": 65536, "kv_heads": 32768}), stream=0, **{**ARGS, "tokens": 0})


def test_workspace_size_between_two_threads():
    """A thread that asks at any moment at which another one's answer is being kept gets the need of its own sizes."""
    class Sizes:
        @staticmethod
        def aidn_sdpa_kv8_workspace_bytes(handle, batch, seq_q, seq_kv):
            return batch * 1000000 + seq_q * 1000 + seq_kv

    class Watched(N.Handle):
        def __init__(self):
            self.__dict__.update(_lib=Sizes, _h=None, _kv8_asked=None, _kv8_sizes=None, _kv8_need=None, other=None)

        def __setattr__(self, name, value):
            object.__setattr__(self, name, value)
            if name != "other" and self.other is None:   # what a thread that runs now would see
                self.other = True
                wrong.extend(s for s in ((1, 2, 3), (4, 5, 6)) if self.kv8_workspace_bytes(*s) != Sizes.aidn_sdpa_kv8_workspace_bytes(None, *s))
                self.other = None

    wrong = []
    h = Watched()
    for sizes in ((1, 2, 3), (4, 5, 6), (1, 2, 3)):
        assert h.kv8_workspace_bytes(*sizes) == Sizes.aidn_sdpa_kv8_workspace_bytes(None, *sizes)
    assert not wrong


def test_append_refuses_a_block_table_between_entries(lib):
    with pytest.raises(N.AidnError) as e:
        N.kv8_append(N.kv8_cache(**{**GOOD, "block_table": 4098}), stream=0, **{**ARGS, "tokens": 0})
    assert "aligned" in str(e.value)


class HostBuffer:
    """What KvCacheFp8 looks at of a GpuBuffer, on the host."""

    def __init__(self, tensor):
        self.tensor, self.Size, self.dtype = tensor, tensor.numel(), tensor.dtype


def test_a_cache_reads_the_buffers_that_it_was_made_with():
    """Neither a buffer nor a size can be put in another's place, and the memory lives as long as the cache does."""
    made = [HostBuffer(torch.zeros(2 * 16 * 2 * 64, dtype=torch.uint8)) for _ in range(2)] + [HostBuffer(torch.ones(4)) for _ in range(2)]
    cache = KvCacheFp8(*made, 16, 2, 64)
    block = cache._pack(4096, 3)
    for name in ("keys", "values", "keyScales", "valueScales", "numBlocks", "blockSize", "kvHeads", "headDim"):
        before = getattr(cache, name)
        with pytest.raises(AttributeError):
            setattr(cache, name, before)
    was = [b.tensor.data_ptr() for b in made]
    held = weakref.ref(made[0].tensor)
    made[0].tensor = torch.zeros_like(made[0].tensor)
    assert held() is not None and cache._pack(4096, 3) == block
    assert list(N._KV8_CACHE.unpack(block)[:4]) == was
