"""Serving from a paged key/value cache held in 8 bits, as measurable cases over the library's public entry points.

Two operators that work on one pool:

  ``append``  rotates a step's queries and keys by their positions, writes the queries out, and puts keys and values into
              their sequences' blocks as E4M3 codes
  ``attend``  attention of a step's queries over what the sequences have in the pool: one token each, a few, or chunks

The pool has [blocks, block size, KV heads, head size] codes for keys and for values, and for each a scale per (block,
head): an element stands for code * scale.  A scale is the smallest power of two (from 2^-100 on) with which no element of the
block is above 448, the largest code.  A block that already holds tokens keeps its scale unless a new token needs a larger
one, for which the codes that it has are moved.

In ``append`` cases the pool has the blocks that the step touches and nothing else, so that all of it can be returned;
what a sequence holds before them is not looked at by the operator.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST_CODE = 448.0


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence behind its projection: launches and latency
        dict(name="append_1_token_h32_kv8_d128", kind="append", dtype="bf16", batch=1, least=1, most=1, heads=32, kv_heads=8,
             dim=128, block=16, before=1236, rope="interleaved", lengths=1),
        # one token of each of 64 sequences, contexts as in the batched decode
        dict(name="append_64_tokens_h32_kv8_d128", kind="append", dtype="bf16", batch=64, least=1, most=1, heads=32,
             kv_heads=8, dim=128, block=16, before=4096, rope="interleaved", lengths=2),
        # prompts of unequal lengths with a head size of 64 and no grouping, pairs half a head apart
        dict(name="append_13_prompts_h16_d64_f16", kind="append", dtype="f16", batch=13, least=97, most=1999, heads=16,
             kv_heads=16, dim=64, block=32, before=700, rope="halves", lengths=3),
        # one long prompt as a whole
        dict(name="append_8192_tokens_h32_kv8_d128", kind="append", dtype="bf16", batch=1, least=8192, most=8192, heads=32,
             kv_heads=8, dim=128, block=16, before=0, rope="interleaved", lengths=4),
        # one token of one sequence, no grouping: launches and latency
        dict(name="attend_1_token_h32_d64_ctx1237", kind="attend", dtype="f16", out="f16", batch=1, least=1, most=1, heads=32,
             kv_heads=32, dim=64, block=16, shortest=1237, longest=1237, softcap=0.0, stats=False, lengths=5),
        # a serving step of sixteen sequences of unequal lengths
        dict(name="attend_16_tokens_h32_kv8_d128_ctx2048", kind="attend", dtype="bf16", out="bf16", batch=16, least=1, most=1,
             heads=32, kv_heads=8, dim=128, block=16, shortest=128, longest=2048, softcap=0.0, stats=False, lengths=6),
        # the batched decode, no grouping: bound by the pool's bytes
        dict(name="attend_64_tokens_h32_d128_ctx4096", kind="attend", dtype="bf16", out="bf16", batch=64, least=1, most=1,
             heads=32, kv_heads=32, dim=128, block=16, shortest=512, longest=4096, softcap=0.0, stats=False, lengths=7),
        # few sequences with long contexts, eight query heads to a KV head, blocks of 64
        dict(name="attend_2_tokens_h64_kv8_d128_ctx32768", kind="attend", dtype="bf16", out="bf16", batch=2, least=1, most=1,
             heads=64, kv_heads=8, dim=128, block=64, shortest=20011, longest=32768, softcap=0.0, stats=False, lengths=8),
        # a step that checks drafted tokens: one to eight queries a sequence, with statistics
        dict(name="attend_drafts_24_h32_kv8_d128_ctx4096", kind="attend", dtype="f16", out="f16", batch=24, least=1, most=8,
             heads=32, kv_heads=8, dim=128, block=16, shortest=200, longest=4096, softcap=0.0, stats=True, lengths=9),
        # single tokens and prompt chunks in one batch, head size 64, blocks of 32, logits capped
        dict(name="attend_mixed_12_h16_kv4_d64_ctx6000", kind="attend", dtype="bf16", out="bf16", batch=12, least=1, most=509,
             heads=16, kv_heads=4, dim=64, block=32, shortest=600, longest=6000, softcap=30.0, stats=False, lengths=10),
        # a large chunk of a long prompt against the cache built so far: bound by arithmetic
        dict(name="attend_2048_at_14336_h32_kv8_d128", kind="attend", dtype="bf16", out="bf16", batch=1, least=2048,
             most=2048, heads=32, kv_heads=8, dim=128, block=16, shortest=16384, longest=16384, softcap=0.0, stats=False,
             lengths=11),
        # queries and results of 32 bits, three queries each, blocks of 24
        dict(name="attend_f32_5x3_h12_kv4_d96_ctx1531", kind="attend", dtype="f32", out="f32", batch=5, least=3, most=3,
             heads=12, kv_heads=4, dim=96, block=24, shortest=3, longest=1531, softcap=0.0, stats=True, lengths=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    dim = rng.choice([64, 64, 128, 128, 128, 96, 256])
    block = rng.choice([8, 16, 16, 16, 32, 64, 24, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 4, 7, 8, 16) if g * kv_heads <= 64])
    lengths = rng.randrange(1 << 20)
    if rng.random() < 0.35:
        batch = _log(rng, 1, 256)
        most = 1 if rng.random() < 0.4 else min(_log(rng, 1, 8192), max(1, 8192 * 32 * 128 // (batch * (heads + 2 * kv_heads) * dim)))
        return dict(kind="append", dtype=dtype, batch=batch, least=rng.choice([1, most, max(1, most // 3)]), most=most, heads=heads,
                    kv_heads=kv_heads, dim=dim, block=block, before=rng.choice([0, _log(rng, 1, 8000)]),
                    rope=rng.choice(["interleaved", "halves"]), lengths=lengths)
    while True:
        batch, longest = _log(rng, 1, 64), _log(rng, 1, 32768)
        most = 1 if rng.random() < 0.5 else min(_log(rng, 1, 2048), longest)
        if batch * longest * kv_heads * dim <= 64 * 4096 * 32 * 128 and batch * heads * most * longest * dim <= 32 * 2048 * 16384 * 128:
            break
    return dict(kind="attend", dtype=dtype, out=dtype, batch=batch, least=rng.choice([1, most]), most=most, heads=heads,
                kv_heads=kv_heads, dim=dim, block=block, shortest=rng.choice([longest, max(1, longest // 7)]), longest=longest,
                softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), stats=rng.choice([True, False]), lengths=lengths)


def _counts(case):
    """(new tokens, tokens in the cache before them) of every sequence: the case's alone, so that its work is known."""
    rng = random.Random(case["lengths"])
    new, before = [], []
    for b in range(case["batch"]):
        n = rng.choice([case["least"], case["most"], _log(rng, case["least"], case["most"])]) if b else case["most"]
        if case["kind"] == "append":
            had = rng.randint(case["before"] // 2, case["before"]) if b else case["before"]
        else:
            had = max(n, rng.randint(case["shortest"], case["longest"]) if b else case["longest"]) - n
        new.append(n)
        before.append(had)
    return new, before


def work(case):
    new, before = _counts(case)
    e, dim, heads, kv_heads, block = BYTES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"], case["block"]
    if case["kind"] == "append":
        tokens = sum(new)
        blocks = sum((a + n - 1) // block - a // block + 1 for n, a in zip(new, before))
        # queries, keys and values in, queries out, codes out, cosines and sines, scales out and those of part-filled blocks in
        moved = tokens * dim * ((2 * heads + 2 * kv_heads) * e + 2 * kv_heads) + tokens * dim * 4
        moved += 8 * kv_heads * (blocks + sum(1 for a in before if a % block))
        return {"bytes": moved, "flops": 3 * tokens * (heads + kv_heads) * dim + 4 * tokens * kv_heads * dim}
    keys = sum(n + a for n, a in zip(new, before))
    blocks = sum(-(-(n + a) // block) for n, a in zip(new, before))
    pairs = sum(n * a + n * (n + 1) // 2 for n, a in zip(new, before))
    moved = 2 * keys * kv_heads * dim + 8 * blocks * kv_heads + sum(new) * heads * (dim * (e + BYTES[case["out"]]) + (4 if case["stats"] else 0))
    return {"bytes": moved, "flops": 4 * dim * heads * pairs}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _scale_of(largest):
    """The power of two for a block whose largest magnitude is `largest`, as a float32 tensor."""
    mantissa, exponent = torch.frexp(largest)           # mantissa in [1/2, 1): 448 is 7/8 of 2^9
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(-100, 119)
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, -100))
    return torch.ldexp(torch.ones_like(largest), exponent)


def _random_pool(blocks, case, generator, device):
    """Codes and scales of `blocks` blocks: normal values, for keys with some channels several times the others."""
    shape = (case["block"], case["kv_heads"], case["dim"])
    codes = torch.empty((blocks,) + shape, dtype=torch.uint8, device=device)
    scales = torch.empty((blocks, case["kv_heads"]), device=device)
    channel = 1 + 3 * (torch.rand(shape[1:], generator=generator, device=device) < 0.05).float()
    step = max(1, (1 << 26) // (shape[0] * shape[1] * shape[2]))
    for at in range(0, blocks, step):
        x = torch.randn((min(step, blocks - at),) + shape, generator=generator, device=device) * channel * 0.5
        s = _scale_of(x.abs().amax((1, 3)))
        scales[at:at + step] = s
        codes[at:at + step] = (x / s[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scales


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    dtype, dim, heads, kv_heads, block, batch = TORCH[case["dtype"]], case["dim"], case["heads"], case["kv_heads"], case["block"], case["batch"]
    new, before = _counts(case)
    tokens, ends = sum(new), [n + a for n, a in zip(new, before)]
    columns = max(-(-e // block) for e in ends)
    first = [a // block if case["kind"] == "append" else 0 for a in before]   # the first block that is in the pool
    counts = [-(-e // block) - f for e, f in zip(ends, first)]
    blocks = sum(counts) + 3
    order = torch.randperm(blocks, generator=g, device=device).to(torch.int32)
    table = torch.zeros((batch, columns), dtype=torch.int32, device=device)
    at = 0
    for b in range(batch):
        table[b, first[b]:first[b] + counts[b]] = order[at:at + counts[b]]
        at += counts[b]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    state = dict(case=case, table=table, columns=columns, tokens=tokens, starts=whole(starts), before=whole(before), ends=whole(ends),
                 uniform=min(new) == max(new))
    state["keys"], state["key_scales"] = _random_pool(blocks, case, g, device)
    state["values"], state["value_scales"] = _random_pool(blocks, case, g, device)
    # for the plain form: each token's sequence and number in it
    state["sequence"] = torch.repeat_interleave(torch.arange(batch, device=device), torch.tensor(new, device=device))
    state["number"] = torch.arange(tokens, device=device) - state["starts"][:-1].long()[state["sequence"]]
    if case["kind"] == "append":
        x = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=g, device=device) * 0.5
        x[:, heads:heads + kv_heads] *= 1 + 3 * (torch.rand((kv_heads, dim), generator=g, device=device) < 0.05).float()
        state["qkv"] = x.to(dtype)
        state["queries"] = torch.empty((tokens, heads, dim), dtype=dtype, device=device)
        angle = torch.arange(max(ends), dtype=torch.float64, device=device)[:, None] * 10000.0 ** (
            -torch.arange(dim // 2, dtype=torch.float64, device=device) * 2 / dim)
        state["cosine"], state["sine"] = angle.cos().float(), angle.sin().float()
    else:
        state["queries"] = (torch.randn((tokens, heads, dim), generator=g, device=device) * 0.5).to(dtype)
        state["out"] = torch.empty((tokens, heads, dim), dtype=TORCH[case["out"]], device=device)
        state["stats"] = torch.empty((tokens, heads), device=device) if case["stats"] else None
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

_backend = None


def _buffers(s):
    """What a program keeps of its tensors: the library's buffer objects and its cache object."""
    from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer, KvCacheFp8
    global _backend
    if _backend is None:
        _backend = CudaBackend(torch.cuda.current_device())
    kept = {k: GpuBuffer(v) for k, v in s.items() if isinstance(v, torch.Tensor) and k not in ("sequence", "number")}
    kept["cache"] = KvCacheFp8(kept["keys"], kept["values"], kept["key_scales"], kept["value_scales"], s["case"]["block"],
                               s["case"]["kv_heads"], s["case"]["dim"])
    return kept


def run(s):
    case = s["case"]
    if not own:
        return _plain_append(s) if case["kind"] == "append" else _plain_attend(s)
    if "kept" not in s:
        s["kept"] = _buffers(s)
    k = s["kept"]
    starts = None if s["uniform"] else k["starts"]
    if case["kind"] == "append":
        _backend.PagedKvAppendFp8(k["qkv"], k["queries"], k["cache"], k["table"], k["before"], case["batch"], s["tokens"],
                                  case["heads"], s["columns"], cos=k["cosine"], sin=k["sine"],
                                  interleaved=case["rope"] == "interleaved", tokenStarts=starts)
        return _append_outputs(s)
    _backend.PagedAttentionFp8(k["queries"], k["cache"], k["table"], k["ends"], k["out"], case["batch"], case["heads"], case["most"],
                               case["longest"], s["columns"], 1 / math.sqrt(case["dim"]), queryStarts=starts,
                               softcap=case["softcap"], softmaxStats=k.get("stats"))
    return _attend_outputs(s)


def _append_outputs(s):
    return dict(queries=s["queries"], keys=s["keys"].view(torch.float8_e4m3fn), values=s["values"].view(torch.float8_e4m3fn),
                key_scales=s["key_scales"], value_scales=s["value_scales"])


def _attend_outputs(s):
    return dict(out=s["out"], stats=s["stats"]) if s["stats"] is not None else dict(out=s["out"])


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    c, s = cos[:, None], sin[:, None]
    pair = (a * c - b * s, a * s + b * c)
    return torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)


def _plain_put(x, codes, scales, block, slot, held):
    """Puts rows x [tokens, heads, dim] into their blocks; `held` [blocks]: how many tokens a block has before them."""
    touched = torch.zeros(len(held), dtype=torch.bool, device=x.device)
    touched[block] = True
    largest = torch.zeros_like(scales)
    largest.scatter_reduce_(0, block[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    had = torch.where((held > 0)[:, None], scales, torch.zeros_like(scales))
    now = torch.where(touched[:, None], torch.maximum(_scale_of(largest), had), scales)
    moved = torch.where((held > 0)[:, None] & touched[:, None], scales / now, torch.ones_like(scales))
    old = (torch.arange(codes.shape[1], device=x.device) < held[:, None])[:, :, None, None] & touched[:, None, None, None]
    again = (codes.view(torch.float8_e4m3fn).float() * moved[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes.copy_(torch.where(old, again, codes))
    codes[block, slot] = (x / now[block][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales.copy_(now)


def _plain_append(s):
    case, heads, kv_heads, size = s["case"], s["case"]["heads"], s["case"]["kv_heads"], s["case"]["block"]
    position = s["before"].long()[s["sequence"]] + s["number"]
    block = s["table"].long()[s["sequence"], position // size]
    held = torch.zeros(len(s["keys"]), dtype=torch.int64, device=block.device)
    part = s["before"].long() // size
    held[s["table"].long()[torch.arange(case["batch"], device=block.device), part.clamp(max=s["columns"] - 1)]] = s["before"].long() % size
    x = s["qkv"].float()
    cos, sin = s["cosine"][position], s["sine"][position]
    both = _rotate(x[:, :heads + kv_heads], cos, sin, case["rope"] == "interleaved")
    s["queries"].copy_(both[:, :heads])
    _plain_put(both[:, heads:], s["keys"], s["key_scales"], block, position % size, held)
    _plain_put(x[:, heads + kv_heads:], s["values"], s["value_scales"], block, position % size, held)
    return _append_outputs(s)


def _plain_attend(s):
    case, batch, kv_heads, dim = s["case"], s["case"]["batch"], s["case"]["kv_heads"], s["case"]["dim"]
    table, most, group = s["table"].long(), s["case"]["most"], s["case"]["heads"] // s["case"]["kv_heads"]
    ends, length = s["ends"].long(), s["table"].shape[1] * s["case"]["block"]

    def rows(codes, scales):   # [batch, heads, keys, dim] in 32 bits
        x = codes.view(torch.float8_e4m3fn)[table].float() * scales[table][:, :, None, :, None]
        return x.reshape(batch, length, kv_heads, dim).transpose(1, 2)

    q = torch.zeros((batch, most) + s["queries"].shape[1:], device=table.device)
    q[s["sequence"], s["number"]] = s["queries"].float()
    q = q.view(batch, most, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, most * group, dim)
    score = q @ rows(s["keys"], s["key_scales"]).transpose(2, 3) * (1 / math.sqrt(dim))
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    last = (ends - new)[:, None] + torch.arange(most, device=table.device)   # the last key that each query sees
    key = torch.arange(length, device=table.device)
    seen = (key <= last[:, :, None]) & (key < ends[:, None, None])
    score.view(batch, kv_heads, most, group, length).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ rows(s["values"], s["value_scales"])) / total.clamp(min=1e-37)
    back = lambda x: x.view(batch, kv_heads, most, group, -1).permute(0, 2, 1, 3, 4).reshape(batch, most, case["heads"], -1)[s["sequence"], s["number"]]  # noqa: E731
    s["out"].copy_(back(out))
    if s["stats"] is not None:
        s["stats"].copy_(back(top + torch.log(total))[..., 0])
    return _attend_outputs(s)


# ---- in 64 bits -----------------------------------------------------------------------------------------------------

def _nearest_code(x):
    """The value of the code nearest to x (64 bits, at most 448): four significant bits, steps of 2^-9 below 2^-6; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    new, before = _counts(case)
    table = s["table"].cpu().tolist()
    heads, kv_heads, dim, size = case["heads"], case["kv_heads"], case["dim"], case["block"]
    starts = s["starts"].cpu().tolist()
    if case["kind"] == "append":
        queries = torch.empty(s["queries"].shape, dtype=torch.float64, device="cuda")
        pools = [[s[n].view(torch.float8_e4m3fn).double(), s[m].double()] for n, m in (("keys", "key_scales"), ("values", "value_scales"))]
        for b, (n, a) in enumerate(zip(new, before)):
            x = s["qkv"][starts[b]:starts[b] + n].double()
            turn = torch.complex(s["cosine"][a:a + n].double(), s["sine"][a:a + n].double())[:, None]
            qk = x[:, :heads + kv_heads]
            if case["rope"] == "interleaved":
                qk = torch.view_as_real(torch.view_as_complex(qk.reshape(n, -1, dim // 2, 2).contiguous()) * turn).reshape(qk.shape)
            else:
                z = torch.complex(qk[..., :dim // 2], qk[..., dim // 2:]) * turn
                qk = torch.cat([z.real, z.imag], -1)
            queries[starts[b]:starts[b] + n] = qk[:, :heads]
            for rows, (values, scales) in zip((qk[:, heads:], x[:, heads + kv_heads:]), pools):
                for j in range(a // size, (a + n - 1) // size + 1):
                    low, high, at = max(a, j * size), min(a + n, (j + 1) * size), table[b][j]
                    part = rows[low - a:high - a]
                    need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((0, 2)) / LARGEST_CODE)).clamp(min=-100))
                    had = low - j * size
                    if had:
                        need = torch.maximum(need, scales[at])
                        values[at, :had] = _nearest_code(values[at, :had] * (scales[at] / need)[:, None])
                    scales[at] = need
                    values[at, had:high - j * size] = _nearest_code(part / need[:, None])
        return dict(queries=queries, keys=pools[0][0], values=pools[1][0], key_scales=pools[0][1], value_scales=pools[1][1])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    stats = torch.zeros(out.shape[:2], dtype=torch.float64, device="cuda")
    for b, (n, a) in enumerate(zip(new, before)):
        at = s["table"][b, :-(-(n + a) // size)].long()
        k, v = (((s[c].view(torch.float8_e4m3fn)[at].double() * s[d][at].double()[:, None, :, None]).reshape(-1, kv_heads, dim)[:n + a])
                for c, d in (("keys", "key_scales"), ("values", "value_scales")))
        hidden = torch.ones((n, n + a), dtype=torch.bool, device="cuda").triu(a + 1)
        for h in range(heads):
            q = s["queries"][starts[b]:starts[b] + n, h].double()
            z = q @ k[:, h // (heads // kv_heads)].T / math.sqrt(dim)
            if case["softcap"]:
                z = torch.tanh(z / case["softcap"]) * case["softcap"]
            z = z.masked_fill(hidden, -math.inf)
            stats[starts[b]:starts[b] + n, h] = torch.logsumexp(z, -1)
            out[starts[b]:starts[b] + n, h] = torch.softmax(z, -1) @ v[:, h // (heads // kv_heads)]
    return dict(out=out, stats=stats) if s["stats"] is not None else dict(out=out)
