"""Rotary positions and linear attention with a decay for each head, as measurable cases over the library's public entry points.

Four operators, as a layer of linear attention uses them:

  ``rotary``    rotates the pairs of a part of each query's and key's head by its position; its gradient is the rotation back
  ``attend``    linear attention of whole sequences: state S_t = exp(g) S_(t-1) + k_t v_t^T, output o_t = scale * q_t S_t
  ``backward``  the gradients of queries, keys, values and of the first states, from those of outputs and last states
  ``step``      one token of each sequence against the states that a server keeps, which it updates

g is a head's log decay (at most 0), a state has [key size, value size] values of 32 bits for each query head.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token behind a packed projection, somewhere in a long context: launches and latency
        dict(name="rotary_1_token_h32_kv8_d128", kind="rotary", dtype="bf16", tokens=1, heads=32, kv_heads=8, dim=128, part=128,
             layout="interleaved", packed=True, back=False, farthest=1 << 20, seq=0, scaling="parts"),
        # a long prompt as a whole
        dict(name="rotary_8192_tokens_h32_kv8_d128", kind="rotary", dtype="bf16", tokens=8192, heads=32, kv_heads=8, dim=128,
             part=128, layout="halves", packed=True, back=False, farthest=8192, seq=0, scaling="none"),
        # the gradient of a training batch, three sequences of odd length, half of each head rotated
        dict(name="rotary_gradient_5997_tokens_h16_d64_f32", kind="rotary", dtype="f32", tokens=5997, heads=16, kv_heads=16, dim=64,
             part=32, layout="halves", packed=False, back=True, farthest=1999, seq=1999, scaling="linear"),
        # one token of one sequence: launches and latency
        dict(name="step_1_h32_d128", kind="step", dtype="bf16", batch=1, heads=32, kv_heads=32, key=128, value=128, decay=True,
             slots=False, lengths=1),
        # one token of each of 64 sequences whose states lie in any order: bound by the states' bytes
        dict(name="step_64_h32_d128", kind="step", dtype="bf16", batch=64, heads=32, kv_heads=32, key=128, value=128, decay=True,
             slots=True, lengths=2),
        # grouped heads, values twice as wide as keys
        dict(name="step_37_h16_kv4_k64_v128_f16", kind="step", dtype="f16", batch=37, heads=16, kv_heads=4, key=64, value=128,
             decay=True, slots=True, lengths=3),
        # a short prompt of odd length that leaves its state
        dict(name="attend_1x517_h16_d64_f16", kind="attend", dtype="f16", batch=1, least=517, most=517, heads=16, kv_heads=16,
             key=64, value=64, decay=True, major="head", ragged="no", first=False, last=True, slots=False, lengths=4),
        # the forward pass of a training step
        dict(name="attend_4x2048_h32_d128", kind="attend", dtype="bf16", batch=4, least=2048, most=2048, heads=32, kv_heads=32,
             key=128, value=128, decay=True, major="head", ragged="no", first=False, last=False, slots=False, lengths=5),
        # prompts of unequal lengths, some of them continued, with grouped heads, as a server takes them
        dict(name="attend_7_prompts_to_8192_h32_kv8_d128", kind="attend", dtype="bf16", batch=7, least=1, most=8192, heads=32,
             kv_heads=8, key=128, value=128, decay=True, major="token", ragged="starts", first=True, last=True, slots=True,
             lengths=6),
        # 32-bit inputs, without a decay
        dict(name="attend_f32_2x1024_h8_d64", kind="attend", dtype="f32", batch=2, least=1024, most=1024, heads=8, kv_heads=8,
             key=64, value=64, decay=False, major="head", ragged="no", first=False, last=True, slots=False, lengths=7),
        # the backward pass of a training step
        dict(name="backward_4x2048_h32_d128", kind="backward", dtype="bf16", batch=4, least=2048, most=2048, heads=32, kv_heads=32,
             key=128, value=128, decay=True, major="head", ragged="no", first=False, last=False, lengths=8),
        # a padded batch with grouped heads and states that carry gradients
        dict(name="backward_3_to_1531_h12_kv4_d64_f16", kind="backward", dtype="f16", batch=3, least=200, most=1531, heads=12,
             kv_heads=4, key=64, value=64, decay=True, major="token", ragged="lengths", first=True, last=True, lengths=9),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "step", "attend", "attend", "backward", "backward"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv_heads <= 64])
    decay = rng.random() < 0.85
    lengths = rng.randrange(1 << 20)
    if kind == "rotary":
        dim = rng.choice([64, 128, 128, 96, 256, 32])
        tokens = _log(rng, 1, min(16384, 4 * 2048 * 32 * 256 // ((heads + kv_heads) * dim)))
        return dict(kind=kind, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    part=rng.choice([dim, dim, dim // 2, dim // 4]), layout=rng.choice(["interleaved", "halves"]),
                    packed=rng.choice([True, False]), back=rng.choice([True, False]), farthest=_log(rng, tokens, 1 << 22),
                    seq=rng.choice([0, tokens, max(1, tokens // 3)]), scaling=rng.choice(["none", "linear", "base", "parts"]))
    key = rng.choice([64, 64, 128, 128, 128, 32, 96, 256])
    value = key if rng.random() < 0.75 else rng.choice([64, 128, 256, 40])
    if kind == "step":
        batch = _log(rng, 1, min(256, max(1, 64 * 32 * 128 * 128 // (heads * key * value))))
        return dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, key=key, value=value, decay=decay,
                    slots=rng.choice([True, False]), lengths=lengths)
    room = max(1, 4 * 2048 * 32 * 128 // (heads * max(key, value)))   # tokens in all
    room = min(room, 16384) // (4 if dtype == "f32" else 1)
    batch = min(_log(rng, 1, 24), max(1, room // 16))
    most = _log(rng, 1, max(1, room // batch))
    case = dict(kind=kind, dtype=dtype, batch=batch, least=rng.choice([1, most, max(1, most // 3)]), most=most, heads=heads,
                kv_heads=kv_heads, key=key, value=value, decay=decay, major=rng.choice(["head", "token"]),
                ragged=rng.choice(["no", "starts", "lengths"]), first=rng.random() < 0.5, last=rng.random() < 0.5)
    if case["ragged"] == "starts":
        case["major"] = "token"
    if case["ragged"] == "no":
        case["least"] = most
    if kind == "attend":
        case["slots"] = (case["first"] and case["last"]) and rng.random() < 0.6
    return dict(case, lengths=lengths)


def _counts(case):
    """The tokens of every sequence: the case's alone, so that its work is known."""
    rng = random.Random(case["lengths"])
    return [rng.choice([case["least"], case["most"], _log(rng, case["least"], case["most"])]) if b else case["most"]
            for b in range(case["batch"])]


def work(case):
    e, heads, kv_heads = BYTES[case["dtype"]], case["heads"], case["kv_heads"]
    if case["kind"] == "rotary":
        n = case["tokens"] * (heads + kv_heads)
        return {"bytes": 2 * n * case["dim"] * e + 4 * case["tokens"] + 4 * case["part"], "flops": 3 * n * case["part"]}
    key, value = case["key"], case["value"]
    tokens = case["batch"] if case["kind"] == "step" else sum(_counts(case))
    states, once = case["batch"] * heads * key * value, tokens * (heads * (key + value) + kv_heads * (key + value)) * e
    if case["kind"] == "step":
        return {"bytes": once + 8 * states, "flops": 5 * states}
    moved = once + 4 * states * (int(case["first"]) + int(case["last"]))
    if case["kind"] == "attend":
        return {"bytes": moved, "flops": 4 * tokens * heads * key * value}
    moved += tokens * e * (heads * key + kv_heads * (key + value)) + 4 * states * int(case["first"])
    return {"bytes": moved, "flops": 10 * tokens * heads * key * value}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _frequencies(case):
    """Radians a position for each pair, in 64 bits, and the factor of the rotated values."""
    half = case["part"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / case["part"])
    if case["scaling"] == "linear":                     # positions compressed eight times
        f = f / 8
    elif case["scaling"] == "base":                     # the base raised, so that the slowest pair turns eight times slower
        f = (10000.0 * 8.0 ** (case["part"] / max(1, case["part"] - 2))) ** (-torch.arange(half, dtype=torch.float64) * 2 / case["part"])
    elif case["scaling"] == "parts":                    # pairs that turn seldom within 4096 positions compressed, fast ones kept
        keep = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f, 0.1 * math.log(8) + 1 if case["scaling"] == "parts" else 1.0


def _decay(case, device):
    """Log decays from -0.7 for the first head to -1/1024 for the last."""
    h = torch.arange(case["heads"], dtype=torch.float64) / max(1, case["heads"] - 1)
    return (-(0.7 ** (1 - h)) * (2.0 ** -10) ** h).float().to(device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    dtype, heads, kv_heads = TORCH[case["dtype"]], case["heads"], case["kv_heads"]

    def normal(*shape, size=0.5, to=dtype):
        return (torch.randn(shape, generator=g, device=device) * size).to(to)

    if case["kind"] == "rotary":
        tokens, dim = case["tokens"], case["dim"]
        f, amplitude = _frequencies(case)
        start = random.Random(seed).randint(0, case["farthest"] - (case["seq"] or tokens))
        at = torch.arange(tokens, device=device) % (case["seq"] or tokens)
        state = dict(case=case, frequencies=f.to(device), amplitude=amplitude, start=start, positions=(start + at).to(torch.int32))
        if case["packed"]:
            state["qkv"] = normal(tokens, heads + 2 * kv_heads, dim, size=1.0)
            state["out"] = torch.empty((tokens, heads + kv_heads, dim), dtype=dtype, device=device)
        else:
            state["q"], state["k"] = normal(tokens, heads, dim, size=1.0), normal(tokens, kv_heads, dim, size=1.0)
            state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
        return state
    key, value, batch = case["key"], case["value"], case["batch"]
    state = dict(case=case, decay=_decay(case, device) if case["decay"] else None)
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    if case["kind"] == "step":
        state |= dict(q=normal(batch, heads, key), k=normal(batch, kv_heads, key), v=normal(batch, kv_heads, value),
                      out=torch.empty((batch, heads, value), dtype=dtype, device=device))
        slots = batch + 3 if case["slots"] else batch
        state["states"] = normal(slots, heads, key, value, to=torch.float32)
        state["slots"] = torch.randperm(slots, generator=g, device=device)[:batch].to(torch.int32) if case["slots"] else None
        return state
    new = _counts(case)
    if case["ragged"] == "starts":
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["starts"] = whole(starts)
        shape = lambda h, d: (sum(new), h, d)  # noqa: E731
    else:
        state["lens"] = whole(new) if case["ragged"] == "lengths" else None
        shape = lambda h, d: (batch, h, case["most"], d) if case["major"] == "head" else (batch, case["most"], h, d)  # noqa: E731
    state |= dict(q=normal(*shape(heads, key)), k=normal(*shape(kv_heads, key)), v=normal(*shape(kv_heads, value)))
    empty = lambda x, to=None: torch.empty_like(x, dtype=to)  # noqa: E731
    if case["kind"] == "backward":
        state["do"] = normal(*shape(heads, value))
        state["first"] = normal(batch, heads, key, value, to=torch.float32) if case["first"] else None
        state["d_last"] = normal(batch, heads, key, value, to=torch.float32) if case["last"] else None
        state["d_first"] = empty(state["first"]) if case["first"] else None
        state |= dict(dq=empty(state["q"]), dk=empty(state["k"]), dv=empty(state["v"]))
        return state
    state["out"] = torch.empty(shape(heads, value), dtype=dtype, device=device)
    slots = batch + 2 if case["slots"] else batch
    state["first"] = normal(slots, heads, key, value, to=torch.float32) if case["first"] else None
    state["last"] = state["first"] if case["slots"] else torch.empty((batch, heads, key, value), device=device) if case["last"] else None
    state["slots"] = torch.randperm(slots, generator=g, device=device)[:batch].to(torch.int32) if case["slots"] else None
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

_backend = None


def _buffers(s):
    """What a program keeps of its tensors: the library's buffer objects."""
    from aidotnet.tensors_b200.backend import CudaBackend, GpuBuffer
    global _backend
    if _backend is None:
        _backend = CudaBackend(torch.cuda.current_device())
    return {k: GpuBuffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}


def run(s):
    case = s["case"]
    if not own:
        return {"rotary": _plain_rotary, "step": _plain_step, "attend": _plain_attend, "backward": _plain_backward}[case["kind"]](s)
    if "kept" not in s:
        s["kept"] = _buffers(s)
    k, heads, kv_heads = s["kept"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotary":
        call = _backend.RotaryEmbeddingBackward if case["back"] else _backend.RotaryEmbedding
        more = dict(interleaved=case["layout"] == "interleaved", amplitude=s["amplitude"])
        more |= dict(seqLen=case["seq"], startPosition=s["start"]) if case["seq"] else dict(positions=k["positions"])
        if case["packed"]:   # the queries and keys of each row are heads side by side
            row = ((heads + 2 * kv_heads) * case["dim"], case["dim"])
            call(k["qkv"], k["out"], None, None, k["frequencies"], case["tokens"], heads + kv_heads, 0, case["dim"], queryStride=row, **more)
        else:
            call(k["q"], k["q_out"], k["k"], k["k_out"], k["frequencies"], case["tokens"], heads, kv_heads, case["dim"], **more)
        return _outputs(s)
    sizes = (case["batch"], heads, kv_heads)
    scale = 1 / math.sqrt(case["key"])
    if case["kind"] == "step":
        _backend.LinearAttentionStep(k["q"], k["k"], k["v"], k["out"], k["states"], k.get("decay"), *sizes, case["key"], case["value"],
                                     scale, stateSlots=k.get("slots"))
        return _outputs(s)
    more = dict(tokenMajor=case["major"] == "token", lengths=k.get("lens"), tokenStarts=k.get("starts"), initialStates=k.get("first"))
    if case["kind"] == "attend":
        _backend.LinearAttention(k["q"], k["k"], k["v"], k["out"], k.get("decay"), *sizes, case["most"], case["key"], case["value"], scale,
                                 finalStates=k.get("last"), stateSlots=k.get("slots"), **more)
    else:
        _backend.LinearAttentionBackward(k["do"], k["q"], k["k"], k["v"], k["dq"], k["dk"], k["dv"], k.get("decay"), *sizes, case["most"],
                                         case["key"], case["value"], scale, gradFinalStates=k.get("d_last"),
                                         gradInitialStates=k.get("d_first"), **more)
    return _outputs(s)


def _outputs(s):
    names = {"rotary": ("out",) if s["case"].get("packed") else ("q_out", "k_out"), "step": ("out", "states"), "attend": ("out", "last"),
             "backward": ("dq", "dk", "dv", "d_first")}[s["case"]["kind"]]
    return {n: s[n] for n in names if s[n] is not None}


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _plain_rotary(s):
    case, part = s["case"], s["case"]["part"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["amplitude"]).float()[:, None], (angle.sin() * s["amplitude"]).float()[:, None]
    if case["back"]:
        sin = -sin

    def turned(x):
        x = x.float()
        y = x[..., :part]
        a, b = (y[..., 0::2], y[..., 1::2]) if case["layout"] == "interleaved" else (y[..., :part // 2], y[..., part // 2:])
        pair = (a * cos - b * sin, a * sin + b * cos)
        y = torch.stack(pair, -1).flatten(-2) if case["layout"] == "interleaved" else torch.cat(pair, -1)
        return torch.cat([y, x[..., part:]], -1)

    if case["packed"]:
        s["out"].copy_(turned(s["qkv"][:, :case["heads"] + case["kv_heads"]]))
    else:
        s["q_out"].copy_(turned(s["q"]))
        s["k_out"].copy_(turned(s["k"]))
    return _outputs(s)


def _log_decay(s):
    return s["decay"] if s["decay"] is not None else torch.zeros(s["case"]["heads"], device=s["q"].device)


def _plain_step(s):
    case, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    k, v = (s[n].float().repeat_interleave(group, 1) for n in ("k", "v"))
    at = s["slots"].long() if s["slots"] is not None else torch.arange(case["batch"], device=k.device)
    now = torch.exp(_log_decay(s))[:, None, None] * s["states"][at] + k[..., :, None] * v[..., None, :]
    s["states"][at] = now
    s["out"].copy_((s["q"].float()[..., None, :] @ now)[..., 0, :] / math.sqrt(case["key"]))
    return _outputs(s)


def _plain_scan(a, b, c, g, x, lag):
    """y_i = exp(g (i + lag)) a_i X + sum over j <= i of exp(g (i - j)) (a_i . b_j) c_j, for [batch, heads, length, size] in
    pieces of 64 whose states come from one product with the pieces' decays; rows past the ends are zeros."""
    batch, heads, length, size = a.shape
    n = 64
    pieces = -(-length // n)
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, pieces * n - length)).view(batch, heads, pieces, n, -1) for t in (a, b, c))
    at = torch.arange(n, device=a.device)
    off = at[:, None] - at
    weight = torch.where(off >= 0, torch.exp(g[:, None, None] * off.clamp(min=0)), torch.zeros((), device=a.device))
    y = ((a @ b.transpose(-1, -2)) * weight[:, None]) @ c
    parts = (b * torch.exp(g[:, None] * (n - 1 - at))[:, None, :, None]).transpose(-1, -2) @ c      # [batch, heads, pieces, size, size]
    p = torch.arange(pieces, device=a.device)
    gap = p[:, None] - p - 1
    carry = torch.where(gap >= 0, torch.exp(g[:, None, None] * (n * gap.clamp(min=0))), torch.zeros((), device=a.device))
    before = (carry @ parts.flatten(3)).view_as(parts)
    y = y + (a * torch.exp(g[:, None] * (at + 1))[:, None, :, None]) @ before
    y = y.view(batch, heads, pieces * n, -1)
    if x is not None:
        step = torch.arange(pieces * n, device=a.device) + lag
        y = y + (a.reshape(batch, heads, pieces * n, size) * torch.exp(g[:, None] * step)[..., None]) @ x
    return y[:, :, :length]


def _plain_rows(s, x, group=1):
    """[batch, heads, length, size] of a tensor in the case's layout, in 32 bits, zeros past a sequence's end."""
    case = s["case"]
    new = _plain_lengths(s)
    at = torch.arange(case["most"], device=x.device)
    if case["ragged"] == "starts":
        x = x[(s["starts"][:-1, None].long() + at).clamp(max=x.shape[0] - 1)].transpose(1, 2)
    elif case["major"] == "token":
        x = x.transpose(1, 2)
    return torch.where((at < new[:, None])[:, None, :, None], x.float(), torch.zeros((), device=x.device)).repeat_interleave(group, 1)


def _plain_back(s, y, to, group=1):
    """Puts [batch, heads, length, size] into a tensor of the case's layout, summed over the heads that share one."""
    case = s["case"]
    y = y.unflatten(1, (-1, group)).sum(2) if group > 1 else y
    inside = torch.arange(case["most"], device=y.device) < _plain_lengths(s)[:, None]
    if case["ragged"] == "starts":
        to.copy_(y.transpose(1, 2)[inside])
    else:
        y = torch.where(inside[:, None, :, None], y, torch.zeros((), device=y.device))
        to.copy_(y if case["major"] == "head" else y.transpose(1, 2))


def _plain_lengths(s):
    if s["case"]["ragged"] == "starts":
        return (s["starts"][1:] - s["starts"][:-1]).long()
    return s["lens"].long() if s["lens"] is not None else torch.full((s["case"]["batch"],), s["case"]["most"], device=s["q"].device)


def _plain_end(b, c, g, new, x, late):
    """The state behind the last token: exp(g n) X + sum over j of exp(g (n - 1 - j + late)) b_j c_j^T."""
    left = (new[:, None] - 1 - torch.arange(b.shape[2], device=b.device)).clamp(min=0)
    y = (b * torch.exp(g[:, None] * (left[:, None] + late))[..., None]).transpose(-1, -2) @ c
    return y if x is None else y + torch.exp(g * new[:, None])[..., None, None] * x


def _plain_attend(s):
    case, group, g = s["case"], s["case"]["heads"] // s["case"]["kv_heads"], _log_decay(s)
    q, k, v = _plain_rows(s, s["q"]), _plain_rows(s, s["k"], group), _plain_rows(s, s["v"], group)
    at = s["slots"].long() if s["slots"] is not None else slice(None)
    first = s["first"][at] if s["first"] is not None else None
    _plain_back(s, _plain_scan(q, k, v, g, first, 1) / math.sqrt(case["key"]), s["out"])
    if s["last"] is not None:
        s["last"][at] = _plain_end(k, v, g, _plain_lengths(s), first, 0)
    return _outputs(s)


def _plain_backward(s):
    case, group, g = s["case"], s["case"]["heads"] // s["case"]["kv_heads"], _log_decay(s)
    scale, new = 1 / math.sqrt(case["key"]), _plain_lengths(s)
    q, do, k, v = _plain_rows(s, s["q"]) * scale, _plain_rows(s, s["do"]), _plain_rows(s, s["k"], group), _plain_rows(s, s["v"], group)
    first = s["first"].transpose(-1, -2) if s["first"] is not None else None
    _plain_back(s, _plain_scan(do, v, k, g, first, 1) * scale, s["dq"])
    # keys and values: the same scan from each sequence's last token to its first
    at = (new[:, None] - 1 - torch.arange(case["most"], device=q.device))
    turn = lambda x: torch.where((at >= 0)[:, None, :, None], x.gather(2, at.clamp(min=0)[:, None, :, None].expand_as(x)), torch.zeros((), device=x.device))  # noqa: E731
    q, do, k, v, last = turn(q), turn(do), turn(k), turn(v), s["d_last"]
    _plain_back(s, turn(_plain_scan(v, do, q, g, last.transpose(-1, -2) if last is not None else None, 0)), s["dk"], group)
    _plain_back(s, turn(_plain_scan(k, q, do, g, last, 0)), s["dv"], group)
    if s["d_first"] is not None:
        s["d_first"].copy_(_plain_end(q, do, g, new, last, 1))
    return _outputs(s)


# ---- in 64 bits -----------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        turn = torch.polar(torch.full_like(s["frequencies"], s["amplitude"]).expand(case["tokens"], -1),
                           s["positions"].double()[:, None] * s["frequencies"] * (-1 if case["back"] else 1))[:, None]

        def rotated(x):
            y, part = x.double(), case["part"]
            z = y[..., :part].unflatten(-1, (-1, 2) if case["layout"] == "interleaved" else (2, -1))
            z = z if case["layout"] == "interleaved" else z.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            y[..., :part] = (z if case["layout"] == "interleaved" else z.transpose(-1, -2)).flatten(-2)
            return y

        if case["packed"]:
            return dict(out=rotated(s["qkv"][:, :case["heads"] + case["kv_heads"]].clone()))
        return dict(q_out=rotated(s["q"].clone()), k_out=rotated(s["k"].clone()))
    heads, group, scale = case["heads"], case["heads"] // case["kv_heads"], 1 / math.sqrt(case["key"])
    rate = [float(x) for x in s["decay"].double().exp()] if s["decay"] is not None else [1.0] * heads
    slots = s["slots"].tolist() if s.get("slots") is not None else list(range(case["batch"]))
    if case["kind"] == "step":
        out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
        states = s["states"].double()
        for b, at in enumerate(slots):
            for h in range(heads):
                states[at, h] = states[at, h] * rate[h] + torch.outer(s["k"][b, h // group].double(), s["v"][b, h // group].double())
                out[b, h] = scale * (states[at, h].T @ s["q"][b, h].double())
        return dict(out=out, states=states)
    new = _counts(case)
    begin = s["starts"].tolist() if case["ragged"] == "starts" else None

    def of(x, b, h):   # rows of one sequence and head
        if begin is not None:
            return x[begin[b]:begin[b + 1], h]
        return x[b, h, :new[b]] if case["major"] == "head" else x[b, :new[b], h]

    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    result = {n: zeros(t) for n, t in _outputs(s).items()}
    if case["kind"] == "attend" and s["slots"] is not None:
        result["last"] = s["first"].double()
    far = torch.arange(max(new), dtype=torch.float64, device="cuda")
    for h in range(heads):
        power = torch.where(far >= 0, torch.tensor(rate[h], dtype=torch.float64, device="cuda") ** far, far)
        for b, n in enumerate(new):
            q, k, v = of(s["q"], b, h).double(), of(s["k"], b, h // group).double(), of(s["v"], b, h // group).double()
            left = (power[:n] * rate[h])[:, None]       # to a row from the state before the first
            rest = power[:n].flip(0)[:, None]           # from a row to the last
            gap = far[:n, None] - far[:n]
            weight = torch.where(gap >= 0, power[gap.clamp(min=0).long()], 0.0) * scale
            if case["kind"] == "attend":
                y = (weight * (q @ k.T)) @ v
                last = k.T @ (rest * v)
                if s["first"] is not None:
                    x = s["first"][slots[b], h].double()
                    y += scale * left * (q @ x)
                    last += rate[h] ** n * x
                of(result["out"], b, h).copy_(y)
                if s["last"] is not None:
                    result["last"][slots[b], h] = last
                continue
            do = of(s["do"], b, h).double()
            d_score = weight * (do @ v.T)
            dq, dk, dv = d_score @ k, d_score.T @ q, (weight * (q @ k.T)).T @ do
            if s["first"] is not None:
                x = s["first"][b, h].double()
                dq += scale * left * (do @ x.T)
                result["d_first"][b, h] = scale * (left * q).T @ do
            if s["d_last"] is not None:
                d = s["d_last"][b, h].double()
                dk += rest * (v @ d.T)
                dv += rest * (k @ d)
                if s["first"] is not None:
                    result["d_first"][b, h] += rate[h] ** n * d
            of(result["dq"], b, h).copy_(dq)
            of(result["dk"], b, h // group).add_(dk)
            of(result["dv"], b, h // group).add_(dv)
    return result
