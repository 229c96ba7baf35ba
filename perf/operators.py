"""What stands around a decode step when a model answers many requests, as timed cases: attention over whole prompts, a
key/value cache held in 4 bits with the attention that reads it, and the log probabilities of the tokens that come out.

  prompt    attention of packed prompts (sequences of different lengths one behind the other), causal, grouped heads
  store     new keys and values into the pages of a 4-bit cache, and the same rows read back as the values they stand for
  cached    attention of each sequence's newest tokens over its pages of the 4-bit cache
  logprobs  log probability of a given token, entropy and the best alternatives of every row of logits

Each is here in its plain form (elementary torch operations in 32 bits) and, where ``own`` is true, as the call that a
program makes of the library. ``listed()`` are the cases that are always timed, ``draw()`` gives others of the same ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DEVICE = "cuda:0"
_GROUP = 32          # channels that share a scale and a lowest value in the 4-bit cache
_LIMIT = 65408.0     # what a value is held to before it is quantized, so that no value read back passes f16's range


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one short request of a small model with one kv head, in single precision: latency counts
        dict(name="prompt_short_f32", kind="prompt", seqs=1, new=77, context=0, heads=4, kv=1, dim=256, window=0, dtype="f32", mix=1),
        # eight requests of different lengths packed into one batch
        dict(name="prompt_packed", kind="prompt", seqs=8, new=1024, context=0, heads=32, kv=8, dim=128, window=0, dtype="f16", mix=2),
        # a long document, every layer global
        dict(name="prompt_long", kind="prompt", seqs=1, new=8192, context=0, heads=32, kv=8, dim=128, window=0, dtype="f16", mix=3),
        # the next piece of a prompt that is taken in pieces: some rows behind a long context, layers that see 512 positions
        dict(name="prompt_piece_local", kind="prompt", seqs=2, new=1000, context=6000, heads=4, kv=1, dim=256, window=512, dtype="f16", mix=4),
        # the new token of each of 48 sequences
        dict(name="store_step", kind="store", seqs=48, new=1, context=2000, kv=8, dim=128, page=64, dtype="f16", mix=5),
        # two whole prompts, from single-precision rows
        dict(name="store_prompt_f32", kind="store", seqs=2, new=8000, context=0, kv=8, dim=128, page=256, dtype="f32", mix=6),
        # one sequence of a small model, one token: latency counts
        dict(name="cached_one_f32", kind="cached", seqs=1, tokens=1, context=2048, heads=4, kv=1, dim=256, window=0, page=2048, dtype="f32", mix=7),
        # twenty requests of very different lengths in small pages, a token of each
        dict(name="cached_ragged", kind="cached", seqs=20, tokens=1, context=8000, heads=32, kv=8, dim=128, window=0, page=16, dtype="f16", mix=8),
        # a few very long contexts, two tokens of each (one of them guessed ahead)
        dict(name="cached_long", kind="cached", seqs=6, tokens=2, context=40000, heads=32, kv=8, dim=128, window=0, page=256, dtype="f16", mix=9),
        # the logits of one decode step of a large vocabulary, with the twenty best
        dict(name="logprobs_step", kind="logprobs", rows=1, vocab=262144, top=20, dtype="f32", banned=0.0),
        # ... of a batch of sequences, half precision, a vocabulary of no round size
        dict(name="logprobs_batch_f16", kind="logprobs", rows=64, vocab=100003, top=5, dtype="f16", banned=0.01),
        # a given text scored: every row's token and entropy
        dict(name="logprobs_score", kind="logprobs", rows=900, vocab=262144, top=1, dtype="f32", banned=0.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(4, 1, 256), (8, 4, 256), (32, 8, 128), (16, 2, 128), (12, 12, 64), (14, 2, 64), (9, 3, 64), (16, 8, 96), (28, 4, 128), (8, 8, 160)]


def draw(rng):
    kind = rng.choices(["prompt", "store", "cached", "logprobs"], [6, 2, 6, 4])[0]
    heads, kv, dim = rng.choice(_HEADS)
    dtype = rng.choice(["f16", "f16", "f32"])
    mix = rng.randrange(1, 1 << 20)
    if kind == "prompt":
        case = dict(kind=kind, seqs=_log_uniform(rng, 1, 16), new=_log_uniform(rng, 8, 8192), context=0, heads=heads, kv=kv, dim=dim,
                    window=0, dtype=dtype, mix=mix)
        if rng.random() < 0.3:
            case["context"] = _log_uniform(rng, 16, 8000)
        if rng.random() < 0.25:
            case["window"] = rng.choice([128, 512, 1000, 1024])
        # what the plain form's scores may take, and single precision costs several times as much
        most = (2.1e9 if dtype == "f16" else 4e8) * min(1.0, 128 / dim)
        while case["seqs"] * heads * case["new"] * (case["new"] + case["context"]) > most:
            if case["seqs"] > 1:
                case["seqs"] -= 1
            else:
                case["new"] = max(1, case["new"] * 7 // 8)
        return case
    if kind == "store":
        case = dict(kind=kind, seqs=_log_uniform(rng, 1, 64), new=rng.choice([1, 1, 2, _log_uniform(rng, 16, 8000)]), context=_log_uniform(rng, 1, 8000),
                    kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype, mix=mix)
        while case["seqs"] * case["new"] * kv * dim > 1.6e7:
            case["new"] = max(1, case["new"] * 3 // 4)
        return case
    if kind == "cached":
        case = dict(kind=kind, seqs=_log_uniform(rng, 1, 64), tokens=rng.choice([1, 1, 1, 2, 4]), context=_log_uniform(rng, 16, 40000), heads=heads, kv=kv,
                    dim=dim, window=rng.choice([0, 0, 0, 512]), page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype, mix=mix)
        while case["seqs"] * case["context"] * max(kv * dim, heads * 16) > 2.4e8:
            if case["seqs"] > 1:
                case["seqs"] -= 1
            else:
                case["context"] = case["context"] * 7 // 8
        return case
    rows = _log_uniform(rng, 1, 900)
    vocab = _log_uniform(rng, 4000, min(262144, 2.35e8 / rows))
    return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20]), dtype=dtype, banned=rng.choice([0.0, 0.01, 0.5]))


# ------------------------------------------------------- lengths and operands

def _lengths(case, longest, least=1):
    """Lengths of a case's sequences: the first is the longest, the others lie anywhere below it."""
    r = random.Random(case["mix"])
    return [longest] + [max(least, _log_uniform(r, max(1, longest // 16), longest)) for _ in range(case["seqs"] - 1)]


def _new_and_all(case):
    """(new rows, rows with the context in front of them) of each sequence."""
    new = _lengths(case, case["new"])
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


def _prepare_prompt(c, g, s):
    new, everything = _new_and_all(c)
    s.new, s.all = new, everything
    s.q_starts, s.k_starts = _ints(_starts(new)), _ints(_starts(everything))
    heads, kv, dim, t = c["heads"], c["kv"], c["dim"], _dtype(c)
    if c["context"]:
        s.q = (1.5 * torch.randn(sum(new), heads, dim, generator=g, device=_DEVICE)).to(t)
        s.k = torch.randn(sum(everything), kv, dim, generator=g, device=_DEVICE).to(t)
        s.v = torch.randn(sum(everything), kv, dim, generator=g, device=_DEVICE).to(t)
    else:
        # queries, keys and values side by side, as one projection leaves them
        rows = torch.randn(sum(new), heads + 2 * kv, dim, generator=g, device=_DEVICE)
        rows[:, :heads] *= 1.5
        rows = rows.to(t)
        s.q, s.k, s.v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    s.y = torch.zeros(sum(new), heads, dim, dtype=t, device=_DEVICE)


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
    s.new, s.all = _new_and_all(c)
    _prepare_pages(c, g, s, s.all)
    s.starts = _ints(_starts(s.new))
    rows = torch.randn(sum(s.new), 2 * c["kv"], c["dim"], generator=g, device=_DEVICE)
    rows[:, :, :: c["dim"] // 2] *= 4.0            # a few channels of every head are larger than the others
    rows = rows.to(_dtype(c))
    s.k, s.v = rows[:, :c["kv"]], rows[:, c["kv"]:]
    s.k_back, s.v_back = (torch.zeros(sum(s.new), c["kv"], c["dim"], dtype=_dtype(c), device=_DEVICE) for _ in range(2))


def _prepare_cached(c, g, s):
    lengths = _lengths(c, max(c["context"], c["tokens"]), c["tokens"])
    s.all = lengths
    _prepare_pages(c, g, s, lengths)
    rows = c["seqs"] * c["tokens"]
    s.q = torch.randn(rows, c["heads"], c["dim"], generator=g, device=_DEVICE).to(_dtype(c))
    s.y = torch.zeros(rows, c["heads"], c["dim"], dtype=_dtype(c), device=_DEVICE)


def _prepare_logprobs(c, g, s):
    rows, vocab = c["rows"], c["vocab"]
    x = 3.0 * torch.randn(rows, vocab, generator=g, device=_DEVICE)
    if c["banned"]:
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device=_DEVICE) < c["banned"], -math.inf)
    s.tokens = torch.randint(0, vocab, (rows,), generator=g, device=_DEVICE, dtype=torch.int32)
    x.scatter_(1, s.tokens.long()[:, None], 6.0)   # the given tokens are likely ones
    s.logits = x.to(_dtype(c))
    s.logprob, s.entropy = (torch.zeros(rows, device=_DEVICE) for _ in range(2))
    s.top_ids = torch.zeros(rows, c["top"], dtype=torch.int32, device=_DEVICE)
    s.top_logprobs = torch.zeros(rows, c["top"], device=_DEVICE)


# ------------------------------------------------------------------- one pass

def run(state):
    if own:
        return globals()["_own_" + state.kind](state)
    return globals()["_plain_" + state.kind](state)


def _own_dtype(s):
    from onnx_vulkan_rs_amd import F16, F32
    return F16 if s.case["dtype"] == "f16" else F32


def _own_heads(s):
    from onnx_vulkan_rs_amd import AttentionHeads
    c = s.case
    return AttentionHeads(n_q_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["dim"], causal=1, window=c["window"], scale=0.0)


def _own_cache(s):
    from onnx_vulkan_rs_amd import Kv4Cache
    c = s.case
    return Kv4Cache(k_codes=s.cache[0].data_ptr(), k_params=s.cache[1].data_ptr(), v_codes=s.cache[2].data_ptr(), v_params=s.cache[3].data_ptr(),
                    n_pages=s.pages, page_size=c["page"], n_kv_heads=c["kv"], head_dim=c["dim"], n_seqs=c["seqs"],
                    lengths=s.lengths.data_ptr(), table=s.table.data_ptr(), table_width=s.width)


def _own_prompt(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import ops
    ops.prompt_attention_device(ctx, _own_heads(s), _own_dtype(s), s.q.data_ptr(), s.q.stride(0), s.k.data_ptr(), s.k.stride(0), s.v.data_ptr(), s.v.stride(0),
                                s.q_starts.data_ptr(), s.k_starts.data_ptr(), len(s.new), s.q.shape[0], s.k.shape[0], s.y.data_ptr(), s.y.stride(0))
    return s.y


def _own_store(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import ops
    cache, dtype, total = _own_cache(s), _own_dtype(s), s.k.shape[0]
    ops.kv4_append_device(ctx, cache, dtype, s.starts.data_ptr(), total, s.k.data_ptr(), s.k.stride(0), s.v.data_ptr(), s.v.stride(0))
    ops.kv4_read_device(ctx, cache, dtype, s.starts.data_ptr(), total, s.k_back.data_ptr(), s.k_back.stride(0), s.v_back.data_ptr(), s.v_back.stride(0))
    return s.k_back, s.v_back


def _own_cached(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import ops
    ops.kv4_attention_device(ctx, _own_cache(s), _own_heads(s), _own_dtype(s), s.case["tokens"], s.q.data_ptr(), s.q.stride(0), s.y.data_ptr(), s.y.stride(0))
    return s.y


def _own_logprobs(s):
    ctx = _context()
    from onnx_vulkan_rs_amd import ops
    top = s.case["top"]
    ops.token_logprobs_device(ctx, _own_dtype(s), s.logits.data_ptr(), s.logits.stride(0), s.logits.shape[0], s.logits.shape[1], s.tokens.data_ptr(),
                              s.logprob.data_ptr(), s.entropy.data_ptr(), top, s.top_ids.data_ptr() if top else None, s.top_logprobs.data_ptr() if top else None)
    return s.logprob, s.entropy, s.top_ids, s.top_logprobs


# --------------------------------------------------------------- plain forms

def _softmax_times(scores, hidden, v):
    """softmax over the last axis of scores (hidden places get nothing) times v; a row with nothing to see is zero."""
    scores = scores.masked_fill_(hidden, -math.inf)
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores.sub_(torch.where(torch.isinf(m), torch.zeros_like(m), m)))
    total = e.sum(-1, keepdim=True)
    n, kv, group, rows, keys = e.shape
    y = torch.bmm(e.reshape(n * kv, group * rows, keys), v).reshape(n, kv, group, rows, -1)
    return y / torch.where(total > 0, total, torch.ones_like(total))


def _padded(rows, starts, longest):
    """Packed rows [total, heads, dim] as [sequences, heads, longest, dim] in 32 bits; what is behind a sequence's end repeats some row."""
    at = (starts[:-1, None].long() + torch.arange(longest, device=rows.device)).clamp_(max=rows.shape[0] - 1)
    return rows[at].float().permute(0, 2, 1, 3)


def _hidden(q_pos, length, keys, window):
    """Which keys a query at position q_pos [sequences, rows] does not see."""
    j = torch.arange(keys, device=q_pos.device)
    gone = (j > q_pos[..., None]) | (j >= length[:, None, None])
    return gone | (j + window <= q_pos[..., None]) if window else gone


def _plain_prompt(s):
    c, n = s.case, len(s.new)
    heads, kv, dim, lq, lk = c["heads"], c["kv"], c["dim"], max(s.new), max(s.all)
    group = heads // kv
    q = _padded(s.q, s.q_starts, lq).reshape(n * kv, group * lq, dim)
    k = _padded(s.k, s.k_starts, lk).reshape(n * kv, lk, dim).transpose(1, 2).contiguous()
    v = _padded(s.v, s.k_starts, lk).reshape(n * kv, lk, dim)
    scores = torch.bmm(q, k).mul_(1.0 / math.sqrt(dim)).reshape(n, kv, group, lq, lk)
    q_len, k_len = (x[1:] - x[:-1] for x in (s.q_starts, s.k_starts))
    q_pos = (k_len - q_len)[:, None] + torch.arange(lq, device=q.device)
    y = _softmax_times(scores, _hidden(q_pos, k_len, lk, c["window"])[:, None, None], v).reshape(n, heads, lq, dim)
    row = torch.arange(s.q.shape[0], device=q.device)
    seq = (row[:, None] >= s.q_starts[1:]).sum(1)
    return y[seq, :, row - s.q_starts[seq]].to(s.q.dtype)


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
    back = []
    for x, codes, params in ((s.k, s.cache[0], s.cache[1]), (s.v, s.cache[2], s.cache[3])):
        # in 64 bits: a quotient next to the border between two codes, or two scales, falls on the side that its exact value has
        g = x.double().clamp(-_LIMIT, _LIMIT).unflatten(-1, (-1, _GROUP))
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        scale, low = ((hi - lo) / 15.0).half(), lo.half()
        steps = (g - low.double()) / torch.where(scale > 0, scale, torch.ones_like(scale)).double()
        code = torch.where(scale > 0, steps, torch.zeros_like(steps)).round().clamp(0, 15).to(torch.uint8).flatten(-2)
        codes[page, :, place] = code[..., 0::2] | (code[..., 1::2] << 4)
        params[page, :, place] = torch.cat([scale, low], -1)
        back.append(_values(codes[page, :, place], params[page, :, place]).to(x.dtype))
    return tuple(back)


def _plain_cached(s):
    c = s.case
    n, tokens, heads, kv, dim = c["seqs"], c["tokens"], c["heads"], c["kv"], c["dim"]
    group, keys = heads // kv, s.width * c["page"]
    k, v = (_values(s.cache[i][s.table.long()], s.cache[i + 1][s.table.long()]).float().transpose(1, 2).reshape(n * kv, keys, dim) for i in (0, 2))
    q = s.q.float().reshape(n, tokens, heads, dim).transpose(1, 2).reshape(n * kv, group * tokens, dim)
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(dim)).reshape(n, kv, group, tokens, keys)
    q_pos = (s.lengths - tokens)[:, None] + torch.arange(tokens, device=q.device)
    y = _softmax_times(scores, _hidden(q_pos, s.lengths, keys, c["window"])[:, None, None], v)
    return y.reshape(n, heads, tokens, dim).transpose(1, 2).reshape(n * tokens, heads, dim).to(s.q.dtype)


def _best(x, top):
    """The ids of the `top` largest of each row, the lower id first among equals: one whole number orders both."""
    bits = (x + 0.0).view(torch.int32).long()                         # (-0 and 0 are equal)
    order = torch.where(bits >= 0, bits, -2147483648 - bits)          # ordered like the floats
    key = (order << 20) | (1048575 - torch.arange(x.shape[1], device=x.device))
    return (1048575 - (key.topk(top, dim=1).values & 1048575)).to(torch.int32)


def _plain_logprobs(s):
    x = s.logits.float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    entropy = lse[:, 0] - torch.where(e > 0, e * x, torch.zeros_like(x)).sum(1) / total[:, 0]
    ids = _best(x, s.case["top"])
    return (x.gather(1, s.tokens.long()[:, None]) - lse)[:, 0], entropy, ids, x.gather(1, ids.long()) - lse


# ------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + s.kind](s)


def _attend_one(q, k, v, first, window):
    """q [heads, rows, dim] at positions first.., k and v [keys, dim] of one kv head, all in 64 bits."""
    pos, j = first + torch.arange(q.shape[1], device=q.device)[:, None], torch.arange(k.shape[0], device=q.device)[None]
    seen = j <= pos
    if window:
        seen &= j > pos - window
    w = torch.where(seen, (q @ k.T) / math.sqrt(q.shape[-1]), -math.inf)
    return torch.nan_to_num(torch.softmax(w, -1)) @ v


def _exact_prompt(s):
    c = s.case
    y = torch.zeros(s.q.shape, dtype=torch.float64, device=_DEVICE)
    group, q_at, k_at = c["heads"] // c["kv"], 0, 0
    for new, everything in zip(s.new, s.all):
        for h in range(c["kv"]):
            k, v = (x[k_at:k_at + everything, h].double() for x in (s.k, s.v))
            for r in range(0, new, 2048):
                n = min(2048, new - r)
                q = s.q[q_at + r:q_at + r + n, h * group:(h + 1) * group].double().transpose(0, 1)
                y[q_at + r:q_at + r + n, h * group:(h + 1) * group] = _attend_one(q, k, v, everything - new + r, c["window"]).transpose(0, 1)
        q_at, k_at = q_at + new, k_at + everything
    return y


def _read64(s, which, seq, first, count):
    """Positions first.. of a sequence from the pages: [kv heads, count, dim]."""
    page = s.case["page"]
    at = torch.arange(first, first + count, device=_DEVICE)
    pages = s.table[seq, at // page].long()
    codes, params = s.cache[which][pages, :, at % page], s.cache[which + 1][pages, :, at % page].double()
    x = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=_DEVICE)
    x[..., 0::2], x[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    scale, low = (params[..., i].repeat_interleave(_GROUP, -1) for i in (0, 1))
    return (low + x * scale).half().double().transpose(0, 1)


def _exact_store(s):
    out = []
    for x in (s.k, s.v):
        g = x.double().clamp(-_LIMIT, _LIMIT).reshape(x.shape[0], x.shape[1], -1, _GROUP)
        lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        scale, low = ((hi - lo) / 15).half().double(), lo.half().double()
        code = torch.round(torch.where(scale > 0, (g - low) / scale, torch.zeros_like(g))).clamp(0, 15)
        out.append((low + code * scale).half().double().reshape(x.shape))
    return tuple(out)


def _exact_cached(s):
    c = s.case
    tokens, group = c["tokens"], c["heads"] // c["kv"]
    y = torch.zeros(s.q.shape, dtype=torch.float64, device=_DEVICE)
    for seq, length in enumerate(s.all):
        k, v = (_read64(s, which, seq, 0, length) for which in (0, 2))
        rows = slice(seq * tokens, (seq + 1) * tokens)
        for h in range(c["kv"]):
            q = s.q[rows, h * group:(h + 1) * group].double().transpose(0, 1)
            y[rows, h * group:(h + 1) * group] = _attend_one(q, k[h], v[h], length - tokens, c["window"]).transpose(0, 1)
    return y


def _exact_logprobs(s):
    out = []
    for r in range(s.logits.shape[0]):
        x = s.logits[r].double()
        logp = torch.log_softmax(x, 0)
        p = logp.exp()
        ids = torch.sort(x, descending=True, stable=True).indices[:s.case["top"]]
        out.append((logp[int(s.tokens[r])], -(p * torch.where(p > 0, logp, torch.zeros_like(p))).sum(), ids.to(torch.int32), logp[ids]))
    return tuple(torch.stack(x) for x in zip(*out))


# ----------------------------------------------------------------------- work

def _seen(new, everything, window):
    """(query, key) pairs of a sequence's causal mask."""
    first = everything - new
    if not window:
        return new * first + new * (new + 1) // 2
    return sum(min(p + 1, window) for p in range(first, everything))


def work(case):
    c = case
    if c["kind"] == "logprobs":
        size = 2 if c["dtype"] == "f16" else 4
        return {"bytes": c["rows"] * (c["vocab"] * size + 12 + 8 * c["top"]), "flops": 5 * c["rows"] * c["vocab"]}
    size, dim, kv = 2 if c["dtype"] == "f16" else 4, c["dim"], c["kv"]
    held = 2 * kv * (dim // 2 + dim // _GROUP * 4)        # bytes of a position in the cache
    if c["kind"] == "prompt":
        new, everything = _new_and_all(c)
        pairs = sum(_seen(n, a, c["window"]) for n, a in zip(new, everything))
        keys = sum(min(a, n + c["window"] - 1) if c["window"] else a for n, a in zip(new, everything))
        return {"bytes": size * dim * (2 * c["heads"] * sum(new) + 2 * kv * keys), "flops": 4 * dim * c["heads"] * pairs}
    if c["kind"] == "store":
        rows = sum(_new_and_all(c)[0])
        return {"bytes": rows * (2 * 2 * kv * dim * size + held), "flops": 8 * rows * kv * dim}
    lengths = _lengths(c, max(c["context"], c["tokens"]), c["tokens"])
    keys = sum(min(a, c["tokens"] + c["window"] - 1) if c["window"] else a for a in lengths)
    pairs = sum(_seen(c["tokens"], a, c["window"]) for a in lengths)
    return {"bytes": keys * held + 2 * c["seqs"] * c["tokens"] * c["heads"] * dim * size, "flops": 4 * dim * c["heads"] * pairs}
