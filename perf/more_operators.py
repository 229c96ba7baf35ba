"""What a layer of a model does with new tokens whose past lies in the paged 4-bit cache, as timed cases: queries and keys normed and
turned by their positions, the same on the way into the cache, and attention of whatever each sequence brings -- a piece of a prompt, a
whole prompt or one token -- over its pages.

  rotary  norms of queries and keys for each head and their rotation by position
  store   the same for rows that go into the cache: queries out, keys and values quantized, and read back as the values they stand for
  chunk   attention of packed new rows, of another number for every sequence, over the pages, with a window and first positions that
          stay visible behind it

Each is here in its plain form (elementary torch operations in 32 bits; angles, and what decides between two codes, in 64) and, where
``own`` is true, as the call that a program makes of the library. ``listed()`` are the cases that are always timed, ``draw()`` gives others
of the same ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DEVICE = "cuda:0"
_GROUP = 32          # channels that share a scale and a lowest value in the 4-bit cache
_LIMIT = 65408.0     # what a value is held to before it is quantized, so that no value read back passes f16's range
_EPS = 1e-6


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the new token of each of 48 sequences: latency counts
        dict(name="rotary_step", kind="rotary", rows=48, heads=32, kv=8, dim=128, turn=128, interleaved=False, norm=True, base=1e6, factor=1, far=20000, dtype="f16"),
        # a long prompt, queries and keys as the projection left them
        dict(name="rotary_prompt", kind="rotary", rows=8192, heads=32, kv=8, dim=128, turn=128, interleaved=False, norm=True, base=1e6, factor=1, far=8192, dtype="f16"),
        # neighbouring channels turned, two thirds of a head, context stretched eightfold, positions far out, no norms, single precision
        dict(name="rotary_far_f32", kind="rotary", rows=1500, heads=16, kv=16, dim=96, turn=64, interleaved=True, norm=False, base=1e4, factor=8, far=1000000, dtype="f32"),
        # the new token of each of 64 sequences into the cache
        dict(name="store_step", kind="store", seqs=64, new=1, context=2000, heads=32, kv=8, dim=128, turn=128, interleaved=False, norm=True, base=1e6, factor=1, page=64, dtype="f16", mix=1),
        # two whole prompts
        dict(name="store_prompt", kind="store", seqs=2, new=6000, context=0, heads=32, kv=8, dim=128, turn=128, interleaved=False, norm=True, base=5e5, factor=4, page=256, dtype="f16", mix=2),
        # a small model with one kv head, in single precision, three requests
        dict(name="store_small_f32", kind="store", seqs=3, new=700, context=100, heads=4, kv=1, dim=256, turn=256, interleaved=False, norm=True, base=1e6, factor=1, page=512, dtype="f32", mix=3),
        # a short follow-up question to a small model: latency counts
        dict(name="chunk_short_f32", kind="chunk", seqs=1, new=77, context=500, ones=0, heads=4, kv=1, dim=256, window=0, sinks=0, page=1024, dtype="f32", mix=4),
        # the next piece of a long document
        dict(name="chunk_long", kind="chunk", seqs=1, new=2048, context=30000, ones=0, heads=32, kv=8, dim=128, window=0, sinks=0, page=256, dtype="f16", mix=5),
        # a serving step: one request's prompt in pieces beside the single tokens of 23 others
        dict(name="chunk_mixed", kind="chunk", seqs=24, new=500, context=8000, ones=23, heads=32, kv=8, dim=128, window=0, sinks=0, page=16, dtype="f16", mix=6),
        # whole prompts of different lengths, stored just before
        dict(name="chunk_prompts", kind="chunk", seqs=6, new=1024, context=0, ones=0, heads=28, kv=4, dim=128, window=0, sinks=0, page=64, dtype="f16", mix=7),
        # pieces of two prompts, a layer that sees 512 positions and the first four
        dict(name="chunk_local", kind="chunk", seqs=2, new=1000, context=6000, ones=0, heads=4, kv=1, dim=256, window=512, sinks=4, page=128, dtype="f16", mix=8),
        # single tokens of long conversations that see the last 4000 positions and the first four
        dict(name="chunk_step_local", kind="chunk", seqs=40, new=1, context=12000, ones=40, heads=32, kv=8, dim=128, window=4000, sinks=4, page=64, dtype="f16", mix=9),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(4, 1, 256), (8, 4, 256), (32, 8, 128), (16, 2, 128), (12, 12, 64), (14, 2, 64), (9, 3, 64), (16, 8, 96), (28, 4, 128), (8, 8, 160)]


def _draw_turn(rng, dim):
    return dict(turn=rng.choice([dim, dim, dim // 2, dim // 32 * 8]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.7, base=rng.choice([1e4, 5e5, 1e6]),
                factor=rng.choice([1, 1, 4, 32]))


def draw(rng):
    kind = rng.choices(["rotary", "store", "chunk"], [3, 3, 8])[0]
    heads, kv, dim = rng.choice(_HEADS)
    dtype = rng.choice(["f16", "f16", "f32"])
    mix = rng.randrange(1, 1 << 20)
    if kind == "rotary":
        rows = _log_uniform(rng, 1, min(8192, 3.3e7 / ((heads + kv) * dim)))
        return dict(kind=kind, rows=rows, heads=heads, kv=kv, dim=dim, far=_log_uniform(rng, 100, 1000000), dtype=dtype, **_draw_turn(rng, dim))
    if kind == "store":
        case = dict(kind=kind, seqs=_log_uniform(rng, 1, 64), new=rng.choice([1, 1, 2, _log_uniform(rng, 16, 6000)]), context=_log_uniform(rng, 1, 8000),
                    heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype, mix=mix, **_draw_turn(rng, dim))
        while case["seqs"] * case["new"] * (heads + 2 * kv) * dim > 5e7:
            case["new"] = max(1, case["new"] * 3 // 4)
        return case
    case = dict(kind=kind, seqs=_log_uniform(rng, 1, 40), new=_log_uniform(rng, 1, 4000), context=rng.choice([0, _log_uniform(rng, 16, 30000)]), ones=0,
                heads=heads, kv=kv, dim=dim, window=rng.choice([0, 0, 128, 1000]), sinks=rng.choice([0, 4, 70]), page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype, mix=mix)
    if not case["window"]:
        case["sinks"] = 0
    if rng.random() < 0.4:
        case["ones"] = rng.randint(0, case["seqs"])
    # what the plain form's scores and gathered pages may take, and single precision costs several times as much
    most = (2.1e9 if dtype == "f16" else 4e8) * min(1.0, 128 / dim)
    while ((case["seqs"] - case["ones"]) * heads * case["new"] * (case["new"] + case["context"]) > most or
           case["seqs"] * (case["new"] + case["context"]) * max(kv * dim, heads * 16) > 2.4e8):
        if case["seqs"] > max(1, case["ones"]):
            case["seqs"] -= 1
        elif case["ones"] > 1:
            case["seqs"], case["ones"] = case["seqs"] - 1, case["ones"] - 1
        else:
            case["new"], case["context"] = max(1, case["new"] * 7 // 8), case["context"] * 7 // 8
    return case


# ------------------------------------------------------- lengths and operands

def _new_and_all(case):
    """(new rows, rows with the context in front of them) of each sequence: the first brings the most, the last ``ones`` one each."""
    r = random.Random(case["mix"])
    longest, n = case["new"], case["seqs"]
    new = [longest] + [max(1, _log_uniform(r, max(1, longest // 16), longest)) for _ in range(n - 1)]
    for s in range(n - case.get("ones", 0), n):
        new[s] = 1
    r = random.Random(case["mix"] + 1)
    before = [case["context"]] + [r.randint(0, case["context"]) for _ in new[1:]]
    return new, [n + b for n, b in zip(new, before)]


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEVICE)


class _State:
    pass


_ctx = None


def _context():
    """The library's context on torch's stream, one per process, as a program keeps it."""
    global _ctx
    if _ctx is None:
        from __graft_entry__ import load_package
        _ctx = load_package().Context(0, stream=torch.cuda.current_stream().cuda_stream)
    return _ctx


def prepare(case, seed):
    s = _State()
    s.kind, s.case = case["kind"], dict(case)
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    globals()["_prepare_" + s.kind](case, g, s)
    return s


def _prepare_turn(c, g, s):
    """The frequencies of a rotation, stretched by parts where the context is longer than the model was trained on (the faster a pair
    turns, the less), and the weights of the norms: what a program keeps with its model."""
    half = c["turn"] // 2
    f = c["base"] ** (-2.0 * torch.arange(half, dtype=torch.float64) / max(1, c["turn"]))
    if c["factor"] > 1:
        keep = ((8192 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        f = f * keep + f / c["factor"] * (1 - keep)
    s.frequencies = f.to(device=_DEVICE, dtype=torch.float32)
    s.amplitude = 1.0 + 0.1 * math.log(c["factor"])
    s.norms = [1 + 0.2 * torch.randn(c["dim"], generator=g, device=_DEVICE) if c["norm"] else None for _ in range(2)]


def _projected(c, g, rows):
    """Queries, keys and values side by side, as one projection leaves them; a few channels of every head are larger than the others."""
    x = torch.randn(rows, c["heads"] + 2 * c["kv"], c["dim"], generator=g, device=_DEVICE)
    x[:, :, :: c["dim"] // 2] *= 4.0
    x = x.to(_dtype(c))
    return x[:, :c["heads"]], x[:, c["heads"]:c["heads"] + c["kv"]], x[:, c["heads"] + c["kv"]:]


def _prepare_rotary(c, g, s):
    _prepare_turn(c, g, s)
    s.q, s.k, _ = _projected(c, g, c["rows"])
    s.positions = torch.randint(0, c["far"], (c["rows"],), generator=g, device=_DEVICE, dtype=torch.int32)
    s.q_out, s.k_out = (torch.zeros(x.shape, dtype=x.dtype, device=_DEVICE) for x in (s.q, s.k))


def _prepare_pages(c, g, s, lengths):
    """A cache of pages in no particular order, some of them nobody's, and which of them are whose."""
    width = -(-max(lengths) // c["page"])
    s.width, s.pages = width, width * len(lengths) + 3
    kv, page, dim = c["kv"], c["page"], c["dim"]
    s.table = torch.randperm(s.pages, generator=g, device=_DEVICE)[:width * len(lengths)].to(torch.int32).reshape(len(lengths), width).contiguous()
    s.lengths = _ints(lengths)
    s.cache = []
    for _ in range(2):
        codes = torch.randint(0, 256, (s.pages, kv, page, dim // 2), generator=g, device=_DEVICE, dtype=torch.uint8)
        params = torch.empty(s.pages, kv, page, dim // _GROUP, 2, dtype=torch.float16, device=_DEVICE)
        params[..., 0] = 0.15 + 0.15 * torch.rand(params.shape[:-1], generator=g, device=_DEVICE)
        params[..., 1] = -8.0 * params[..., 0] + 0.2 * torch.randn(params.shape[:-1], generator=g, device=_DEVICE)
        s.cache += [codes, params]


def _prepare_store(c, g, s):
    _prepare_turn(c, g, s)
    s.new, s.all = _new_and_all(c)
    _prepare_pages(c, g, s, s.all)
    s.starts = _ints(_starts(s.new))
    s.q, s.k, s.v = _projected(c, g, sum(s.new))
    s.q_out = torch.zeros(s.q.shape, dtype=s.q.dtype, device=_DEVICE)
    s.k_back, s.v_back = (torch.zeros(s.k.shape, dtype=torch.float16, device=_DEVICE) for _ in range(2))


def _prepare_chunk(c, g, s):
    s.new, s.all = _new_and_all(c)
    _prepare_pages(c, g, s, s.all)
    s.starts = _ints(_starts(s.new))
    s.q = (1.5 * torch.randn(sum(s.new), c["heads"], c["dim"], generator=g, device=_DEVICE)).to(_dtype(c))
    s.y = torch.zeros(s.q.shape, dtype=s.q.dtype, device=_DEVICE)
    # the sequences that bring a few rows and those that bring many, each padded to the longest of its kind by the plain form
    few = [i for i, n in enumerate(s.new) if n <= 16]
    many = [i for i, n in enumerate(s.new) if n > 16]
    s.kinds = [(torch.tensor(x, device=_DEVICE), max(s.new[i] for i in x)) for x in (few, many) if x]


# ------------------------------------------------------------------- one pass

def run(state):
    if own:
        return globals()["_own_" + state.kind](state)
    return globals()["_plain_" + state.kind](state)


def _own_dtype(s):
    from onnx_vulkan_rs_amd import F16, F32
    return F16 if s.case["dtype"] == "f16" else F32


def _own_rotary_heads(s):
    from onnx_vulkan_rs_amd import RotaryHeads
    c = s.case
    q_norm, k_norm = (x.data_ptr() if x is not None else None for x in s.norms)
    return RotaryHeads(n_q_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["dim"], rotary_dim=c["turn"], interleaved=int(c["interleaved"]), norm_eps=_EPS,
                       amplitude=s.amplitude, frequencies=s.frequencies.data_ptr(), q_norm=q_norm, k_norm=k_norm)


def _own_cache(s):
    from onnx_vulkan_rs_amd import Kv4Cache
    c = s.case
    return Kv4Cache(k_codes=s.cache[0].data_ptr(), k_params=s.cache[1].data_ptr(), v_codes=s.cache[2].data_ptr(), v_params=s.cache[3].data_ptr(),
                    n_pages=s.pages, page_size=c["page"], n_kv_heads=c["kv"], head_dim=c["dim"], n_seqs=c["seqs"],
                    lengths=s.lengths.data_ptr(), table=s.table.data_ptr(), table_width=s.width)


def _own_rotary(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import ops
    ops.rotary_device(ctx, _own_rotary_heads(s), _own_dtype(s), s.positions.data_ptr(), s.q.shape[0], s.q.data_ptr(), s.q.stride(0), s.k.data_ptr(), s.k.stride(0),
                      s.q_out.data_ptr(), s.q_out.stride(0), s.k_out.data_ptr(), s.k_out.stride(0))
    return s.q_out, s.k_out


def _own_store(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import F16, ops
    cache, total = _own_cache(s), s.k.shape[0]
    ops.kv4_append_rotary_device(ctx, cache, _own_rotary_heads(s), _own_dtype(s), s.starts.data_ptr(), total, s.q.data_ptr(), s.q.stride(0), s.k.data_ptr(), s.k.stride(0),
                                 s.v.data_ptr(), s.v.stride(0), s.q_out.data_ptr(), s.q_out.stride(0))
    ops.kv4_read_device(ctx, cache, F16, s.starts.data_ptr(), total, s.k_back.data_ptr(), s.k_back.stride(0), s.v_back.data_ptr(), s.v_back.stride(0))
    return s.q_out, s.k_back, s.v_back


def _own_chunk(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import AttentionHeads, ops
    c = s.case
    heads = AttentionHeads(n_q_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["dim"], causal=1, window=c["window"], scale=0.0)
    ops.kv4_prompt_attention_device(ctx, _own_cache(s), heads, c["sinks"], _own_dtype(s), s.starts.data_ptr(), s.q.shape[0], s.q.data_ptr(), s.q.stride(0),
                                    s.y.data_ptr(), s.y.stride(0))
    return s.y


# --------------------------------------------------------------- plain forms

def _turned(s, x, norm, positions):
    """Rows of heads [rows, heads, dim] normed and turned, in 32 bits and rounded once; angles in 64."""
    c, half = s.case, s.case["turn"] // 2
    y = x.float()
    if norm is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * norm
    angle = positions.double()[:, None] * s.frequencies.double()
    cos, sin = (f(angle).float()[:, None] * s.amplitude for f in (torch.cos, torch.sin))
    if c["interleaved"]:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_rotary(s):
    return _turned(s, s.q, s.norms[0], s.positions), _turned(s, s.k, s.norms[1], s.positions)


def _values(codes, params):
    """What codes stand for: each rounded once to f16."""
    x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    x = x.unflatten(-1, (-1, _GROUP)) * params[..., :1].float() + params[..., 1:].float()
    return x.flatten(-2).half()


def _plain_store(s):
    c, total = s.case, s.k.shape[0]
    row = torch.arange(total, device=s.k.device)
    seq = (row[:, None] >= s.starts[1:]).sum(1)
    pos = s.lengths[seq] - (s.starts[seq + 1] - s.starts[seq]) + row - s.starts[seq]
    page, place = s.table[seq, pos // c["page"]].long(), pos % c["page"]
    q, k = _turned(s, s.q, s.norms[0], pos), _turned(s, s.k, s.norms[1], pos)
    back = []
    for x, codes, params in ((k, s.cache[0], s.cache[1]), (s.v, s.cache[2], s.cache[3])):
        # in 64 bits: a quotient next to the border between two codes, or two scales, falls on the side that its exact value has
        g = x.double().clamp(-_LIMIT, _LIMIT).unflatten(-1, (-1, _GROUP))
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        scale, low = ((hi - lo) / 15.0).half(), lo.half()
        steps = (g - low.double()) / torch.where(scale > 0, scale, torch.ones_like(scale)).double()
        code = torch.where(scale > 0, steps, torch.zeros_like(steps)).round().clamp(0, 15).to(torch.uint8).flatten(-2)
        codes[page, :, place] = code[..., 0::2] | (code[..., 1::2] << 4)
        params[page, :, place] = torch.cat([scale, low], -1)
        back.append(_values(codes[page, :, place], params[page, :, place]))
    return q, back[0], back[1]


def _softmax_times(scores, hidden, v):
    """softmax over the last axis of scores (hidden places get nothing) times v; a row with nothing to see is zero."""
    scores = scores.masked_fill_(hidden, -math.inf)
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores.sub_(torch.where(torch.isinf(m), torch.zeros_like(m), m)))
    total = e.sum(-1, keepdim=True)
    n, kv, group, rows, keys = e.shape
    y = torch.bmm(e.reshape(n * kv, group * rows, keys), v).reshape(n, kv, group, rows, -1)
    return y / torch.where(total > 0, total, torch.ones_like(total))


def _plain_kind(s, seqs, longest):
    """The rows of some sequences, padded to the longest: which rows of them there are, and their results."""
    c = s.case
    heads, kv, dim, n, keys = c["heads"], c["kv"], c["dim"], seqs.shape[0], s.width * c["page"]
    group, table = heads // kv, s.table[seqs].long()
    k, v = (_values(s.cache[i][table], s.cache[i + 1][table]).float().transpose(1, 2).reshape(n * kv, keys, dim) for i in (0, 2))
    first, count, length = s.starts[seqs].long(), (s.starts[seqs + 1] - s.starts[seqs]).long(), s.lengths[seqs].long()
    step = torch.arange(longest, device=seqs.device)
    at = (first[:, None] + step).clamp_(max=s.q.shape[0] - 1)
    q = s.q[at].float().permute(0, 2, 1, 3).reshape(n * kv, group * longest, dim)
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(dim)).reshape(n, kv, group, longest, keys)
    pos, j = (length - count)[:, None] + step, torch.arange(keys, device=seqs.device)
    hidden = (j > pos[..., None]) | (j >= length[:, None, None])
    if c["window"]:
        hidden |= (j + c["window"] <= pos[..., None]) & (j >= c["sinks"])
    y = _softmax_times(scores, hidden[:, None, None], v).reshape(n, heads, longest, dim).transpose(1, 2)
    there = step < count[:, None]
    return at[there], y[there]


def _plain_chunk(s):
    y = torch.zeros_like(s.q)
    for rows, values in (_plain_kind(s, *kind) for kind in s.kinds):
        y[rows] = values.to(y.dtype)
    return y


# ------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + s.kind](s)


def _turn64(s, x, norm, positions):
    half = s.case["turn"] // 2
    y = x.double()
    if norm is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + _EPS) * norm.double()
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if s.case["interleaved"] else (i, i + half)
    turn = s.amplitude * torch.exp(1j * positions.double().outer(s.frequencies.double()))
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(s):
    return _turn64(s, s.q, s.norms[0], s.positions), _turn64(s, s.k, s.norms[1], s.positions)


def _exact_store(s):
    pos = torch.cat([torch.arange(a - n, a, device=_DEVICE) for n, a in zip(s.new, s.all)])
    q, k = _turn64(s, s.q, s.norms[0], pos), _turn64(s, s.k, s.norms[1], pos)
    out = [q]
    for x in (k.to(s.k.dtype), s.v):       # (keys are rows of the type on their way into the cache)
        g = x.double().clamp(-_LIMIT, _LIMIT).reshape(x.shape[0], x.shape[1], -1, _GROUP)
        lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        scale, low = ((hi - lo) / 15).half().double(), lo.half().double()
        code = torch.round(torch.where(scale > 0, (g - low) / scale, torch.zeros_like(g))).clamp(0, 15)
        out.append((low + code * scale).half().double().reshape(x.shape))
    return tuple(out)


def _attend_one(q, k, v, first, window, sinks):
    """q [heads, rows, dim] at positions first.., k and v [keys, dim] of one kv head, all in 64 bits."""
    pos, j = first + torch.arange(q.shape[1], device=q.device)[:, None], torch.arange(k.shape[0], device=q.device)[None]
    seen = j <= pos
    if window:
        seen &= (j > pos - window) | (j < sinks)
    w = torch.where(seen, (q @ k.T) / math.sqrt(q.shape[-1]), -math.inf)
    return torch.nan_to_num(torch.softmax(w, -1)) @ v


def _read64(s, which, seq, count):
    """The first positions of a sequence from the pages: [kv heads, count, dim]."""
    page = s.case["page"]
    at = torch.arange(count, device=_DEVICE)
    pages = s.table[seq, at // page].long()
    codes, params = s.cache[which][pages, :, at % page], s.cache[which + 1][pages, :, at % page].double()
    x = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=_DEVICE)
    x[..., 0::2], x[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    scale, low = (params[..., i].repeat_interleave(_GROUP, -1) for i in (0, 1))
    return (low + x * scale).half().double().transpose(0, 1)


def _exact_chunk(s):
    c = s.case
    y = torch.zeros(s.q.shape, dtype=torch.float64, device=_DEVICE)
    group, at = c["heads"] // c["kv"], 0
    for seq, (new, length) in enumerate(zip(s.new, s.all)):
        k, v = (_read64(s, which, seq, length) for which in (0, 2))
        for h in range(c["kv"]):
            for r in range(0, new, 1024):
                n = min(1024, new - r)
                q = s.q[at + r:at + r + n, h * group:(h + 1) * group].double().transpose(0, 1)
                y[at + r:at + r + n, h * group:(h + 1) * group] = _attend_one(q, k[h], v[h], length - new + r, c["window"], c["sinks"]).transpose(0, 1)
        at += new
    return y


# ----------------------------------------------------------------------- work

def _seen(new, everything, window, sinks):
    """(query, key) pairs of a sequence's mask."""
    first = everything - new
    if not window:
        return new * first + new * (new + 1) // 2
    return sum(min(p + 1, window) + min(max(0, p + 1 - window), sinks) for p in range(first, everything))


def work(case):
    c = case
    size, dim, kv, heads = 2 if c["dtype"] == "f16" else 4, c["dim"], c["kv"], c["heads"]
    held = 2 * kv * (dim // 2 + dim // _GROUP * 4)        # bytes of a position in the cache
    if c["kind"] == "rotary":
        return {"bytes": c["rows"] * (4 + 2 * size * (heads + kv) * dim), "flops": c["rows"] * (heads + kv) * (3 * c["turn"] + (4 * dim if c["norm"] else 0))}
    if c["kind"] == "store":
        rows = sum(_new_and_all(c)[0])
        return {"bytes": rows * (size * dim * (2 * heads + 2 * kv) + held + 2 * 2 * dim * kv), "flops": rows * ((heads + kv) * (3 * c["turn"] + 4 * dim) + 16 * kv * dim)}
    new, everything = _new_and_all(c)
    pairs = sum(_seen(n, a, c["window"], c["sinks"]) for n, a in zip(new, everything))
    keys = sum(min(a, n + c["window"] - 1 + c["sinks"]) if c["window"] else a for n, a in zip(new, everything))
    return {"bytes": keys * held + 2 * sum(new) * heads * dim * size, "flops": 4 * dim * heads * pairs}
