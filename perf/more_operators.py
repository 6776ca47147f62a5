"""What the operators of a paged cache of keys and values are measured on: rotary positions (forward
and backward), appending keys and values to the cache with the rotation on the way, and attention of
new queries against the cache, with a prefix that the whole batch shares.

A cache holds pages of `page` tokens, in fp32, bf16 or e4m3 with an fp32 scale for each row (a token's
head). A batch is `seqs` sequences; sequence s has the rows starts[s] .. starts[s + 1] - 1 of q, k, v
and the output, and lengths[s] keys of its own with those rows' included, in the pages that its row of
the table names. A shared prefix lies in pages of its own, in front of every sequence. With `own` false
`run` computes in elementary torch operations; with `own` true it makes the framework's calls on the
same tensors.

Kinds of case and the ranges that `draw` takes them from:
* rope    1 .. 16384 rows of 1 .. 40 heads of 32 .. 128, all of a head or part of it turned, halves or
          neighbours paired, steps scaled for long contexts or not, forward or backward;
* append  1 .. 256 sequences, up to 2048 new tokens each and 16384 in all, 1 .. 16 heads of 64 .. 128;
* attend  1 .. 256 sequences of up to 8192 keys, 1 .. 512 queries each, 1 .. 8 query heads for each of
          1 .. 8 heads of 64 .. 128, with no prefix or one of 256 .. 16384 keys.
"""
import math

import torch

own = False

BASE = 10000.0
TOP = 448.0        # the largest e4m3 value
FAR = 131072       # positions of rope
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}


def _rope(tokens, heads, d, rot, interleaved=False, scaled=False, backward=False):
    return dict(kind="rope", tokens=tokens, heads=heads, d=d, rot=rot, interleaved=interleaved,
                scaled=scaled, backward=backward)


def _append(seqs, new, heads, d, held, page, rot, q_heads=0, interleaved=False, behind=0):
    return dict(kind="append", seqs=seqs, least=1 if behind else new, new=new, heads=heads, d=d,
                held=held, page=page, rot=rot, q_heads=q_heads, interleaved=interleaved,
                behind=behind)


def _attend(seqs, low, high, new, heads, group, d, held, page, prefix=0, ragged=False, behind=0):
    return dict(kind="attend", seqs=seqs, low=low, high=high, least=1 if ragged else new, new=new,
                heads=heads, group=group, d=d, held=held, page=page, prefix=prefix, behind=behind)


def listed():
    return [
        # The queries and keys of a decoding step of 64 sequences: latency.
        dict(name="rope_step", **_rope(64, 40, 128, 128)),
        # A ragged batch whose heads turn in part, neighbours paired, steps scaled for a long context.
        dict(name="rope_part", **_rope(4093, 17, 80, 48, interleaved=True, scaled=True)),
        # The gradient of a long prompt's queries and keys.
        dict(name="rope_backward", **_rope(16384, 40, 128, 128, backward=True)),
        # A decoding step: one new key and value for each of 64 sequences, in 8 bits; the queries are
        # turned by the same call.
        dict(name="append_step", **_append(64, 1, 8, 128, "e4m3", 16, 128, q_heads=32)),
        # Ragged pieces of prompts into an fp32 cache, with padding rows behind them.
        dict(name="append_ragged", **_append(37, 300, 5, 80, "f32", 32, 48, interleaved=True,
                                             behind=7)),
        # Eight long prompts into a bf16 cache.
        dict(name="append_prompt", **_append(8, 2048, 8, 128, "bf16", 64, 128)),
        # One sequence, one query: latency.
        dict(name="attend_one", **_attend(1, 4096, 4096, 1, 8, 4, 128, "bf16", 16)),
        # A decoding step of 64 sequences of all lengths, cache in 8 bits.
        dict(name="attend_step", **_attend(64, 97, 8191, 1, 8, 4, 128, "e4m3", 64)),
        # A few queries each (drafted tokens that are checked) in fp32, an empty sequence among them,
        # padding rows behind.
        dict(name="attend_drafts", **_attend(37, 0, 1999, 5, 5, 4, 80, "f32", 16, ragged=True,
                                             behind=3)),
        # Pieces of long prompts against what is cached of them.
        dict(name="attend_pieces", **_attend(4, 2048, 8192, 512, 8, 4, 128, "bf16", 64)),
        # 64 sequences that share instructions of 8192 tokens.
        dict(name="attend_shared", **_attend(64, 33, 511, 1, 8, 4, 128, "bf16", 16, prefix=8192)),
        # 256 sequences that share a document, cache in 8 bits.
        dict(name="attend_document", **_attend(256, 65, 1023, 1, 8, 4, 128, "e4m3", 64,
                                               prefix=16383)),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend"])
    if kind == "rope":
        d = rng.choice([32, 64, 80, 96, 112, 128])
        rot = d if rng.random() < 0.6 else 2 * rng.randint(4, d // 2)
        return _rope(_log(rng, 1, 16384), rng.randint(1, 40), d, rot, rng.random() < 0.5,
                     rng.random() < 0.5, rng.random() < 0.4)
    d = rng.choice([64, 80, 96, 112, 128])
    held = rng.choice(["f32", "bf16", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    seqs = _log(rng, 1, 256)
    if kind == "append":
        new = _log(rng, 1, min(2048, 16384 // seqs))
        heads = rng.randint(1, 16)
        return _append(seqs, new, heads, d, held, page,
                       rng.choice([0, 2 * rng.randint(4, d // 2), d]),
                       q_heads=heads * rng.choice([0, 1, 4]), interleaved=rng.random() < 0.5,
                       behind=rng.choice([0, 0, 5]))
    heads, group = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 8])
    new = 1 if rng.random() < 0.5 else _log(rng, 2, min(512, max(2, 4096 // seqs)))
    # No more scores than 512 queries of 4 sequences have against 8192 keys, no more keys than 64
    # sequences of 8192.
    high = min(8192, (4 << 24) // (seqs * new * 8), 64 * 8192 // seqs)
    high = _log(rng, min(high, max(new, 16)), high)
    prefix = 0 if rng.random() < 0.5 else _log(rng, 256, min(16384, (256 << 14) // (seqs * new)))
    return _attend(seqs, rng.randint(0, high), high, new, heads, group, d, held, page, prefix,
                   ragged=rng.random() < 0.5, behind=rng.choice([0, 0, 3]))


# ---- inputs -------------------------------------------------------------------------------------


def _spread(low, high, count):
    """`count` whole numbers, evenly from low to high."""
    return [low + (high - low) * i // max(1, count - 1) if count > 1 else high for i in range(count)]


def _counts(case):
    """(rows, own keys) of each sequence."""
    rows = _spread(case["least"], case["new"], case["seqs"])
    if case["kind"] == "append":
        return [(n, n + 37 * (i % 3)) for i, n in enumerate(rows)]
    keys = _spread(case["low"], case["high"], case["seqs"])
    # Rows fall, then rise, as the keys grow: the two are not in step.
    return list(zip(rows[1::2][::-1] + rows[0::2], keys))


def _rows_to_e4m3(x):
    """e4m3 values and the scale of each row: max(largest magnitude / 448, 2^-126)."""
    scale = (x.abs().amax(-1) / TOP).clamp_min(2.0 ** -126)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _held(case, gen, pages, filled):
    """A cache of [pages, page, heads, d] (tokens of a page next to each other in fp32 and bf16) or
    [pages, heads, page, d] (8 bits, with scales [pages, heads, page]); empty pages are zeros."""
    heads, d, page = case["heads"], case["d"], case["page"]
    out = {}
    for name in ("k", "v"):
        shape = (pages, heads, page, d) if case["held"] == "e4m3" else (pages, page, heads, d)
        x = torch.randn(shape, generator=gen, device="cuda") if filled else torch.zeros(
            shape, device="cuda")
        if filled and name == "k":
            x = x * torch.exp(0.4 * torch.randn((d,), generator=gen, device="cuda"))
        if case["held"] == "e4m3":
            out[name], out[name + "_scales"] = _rows_to_e4m3(x)
        else:
            out[name] = x.to(DTYPES[case["held"]])
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def whole(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    d = case["d"]
    if case["kind"] == "rope":
        state["x"] = normal(case["tokens"], case["heads"], d)
        state["positions"] = torch.randint(0, FAR, (case["tokens"],), generator=gen, device="cuda",
                                           dtype=torch.int32)
        state["out"] = torch.zeros_like(state["x"])
        return state
    host = torch.Generator().manual_seed(seed)
    counts = _counts(case)
    counts = [counts[i] for i in torch.randperm(len(counts), generator=host).tolist()]
    starts = [0]
    for n, _ in counts:
        starts.append(starts[-1] + n)
    rows = starts[-1] + case["behind"]
    page, prefix = case["page"], case.get("prefix", 0)
    used = [-(-keys // page) for _, keys in counts]
    width = max(1, max(used))
    shared = -(-prefix // page)
    order = torch.randperm(sum(used) + shared, generator=host).tolist()
    pages, at = [], shared
    for n in used:
        pages.append(order[at:at + n] + [0] * (width - n))
        at += n
    state["starts"], state["lengths"] = whole(starts), whole([keys for _, keys in counts])
    state["pages"] = whole(pages)
    if prefix:
        state["prefix_pages"] = whole(order[:shared])
    total = max(1, len(order))
    state.update(_held(case, gen, total, case["kind"] == "attend"))
    if case["kind"] == "append":
        state["new_k"], state["new_v"] = normal(rows, case["heads"], d), normal(rows, case["heads"], d)
        if case["q_heads"]:
            state["q"] = normal(rows, case["q_heads"], d)
            state["q_out"] = torch.zeros_like(state["q"])
    else:
        state["q"] = normal(rows, case["heads"] * case["group"], d)
        state["out"] = torch.zeros_like(state["q"])
    return state


# ---- the plain forms ----------------------------------------------------------------------------


def _scaling(case):
    """Steps divided by 8, but for pairs that turn more than 32 times in 4096 positions; between 1
    and 32 turns by degrees. The amplitude grows with the logarithm."""
    return (dict(factor=8.0, original=4096.0, slow=1.0, fast=32.0),
            0.1 * math.log(8.0) + 1.0) if case.get("scaled") else (dict(), 1.0)


def _steps(case):
    """Radians that each pair turns by from one position to the next, in 64 bits."""
    rot = case["rot"]
    steps = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    scaling, _ = _scaling(case)
    if scaling:
        turns = scaling["original"] * steps / (2 * math.pi)
        kept = ((turns - scaling["slow"]) / (scaling["fast"] - scaling["slow"])).clamp(0, 1)
        steps = steps * (kept + (1 - kept) / scaling["factor"])
    return steps


def _turned(case, x, positions, backward=False):
    """x [rows, heads, d] with its leading `rot` columns turned by its row's angles."""
    rot = case["rot"]
    if rot == 0:
        return x
    angles = positions.double()[:, None, None] * _steps(case)
    _, amplitude = _scaling(case)
    cos, sin = (amplitude * angles.cos()).float(), (amplitude * angles.sin()).float()
    if backward:
        sin = -sin
    head = x[..., :rot]
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((head, x[..., rot:]), -1)


def _places(state, rows):
    """Of each row: its sequence, its place among the sequence's rows and keys, and whether it has a
    sequence."""
    starts, lengths = state["starts"].long(), state["lengths"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    real = seq < lengths.numel()
    seq = seq.clamp_max(lengths.numel() - 1)
    nth = row - starts[seq]
    return seq, nth, lengths[seq] - (starts[seq + 1] - starts[seq]) + nth, real


def _plain_append(state):
    case = state["case"]
    page = case["page"]
    seq, _, place, real = _places(state, state["new_k"].shape[0])
    n = int(case["behind"])
    kept = slice(0, place.numel() - n)
    at = state["pages"].long()[seq, torch.where(real, place // page, 0)][kept]
    off = (place % page)[kept]
    for name in ("k", "v"):
        x = state["new_" + name]
        x = (_turned(case, x, place) if name == "k" else x)[kept]
        if case["held"] == "e4m3":
            values, scale = _rows_to_e4m3(x)
            state[name].view(torch.uint8)[at, :, off] = values.view(torch.uint8)
            state[name + "_scales"][at, :, off] = scale
        else:
            state[name][at, off] = x.to(state[name].dtype)
    if "q" in state:
        state["q_out"][kept] = _turned(case, state["q"], place)[kept]


def _read(state, name, pages, dtype=torch.float32):
    """The rows of the pages, [..., heads, keys, d]."""
    x = state[name].to(dtype)[pages] if state[name].dtype == torch.float32 else state[name].view(
        torch.uint8 if state[name].element_size() == 1 else torch.int16)[pages].view(
            state[name].dtype).to(dtype)
    if state["case"]["held"] == "e4m3":
        x = x * state[name + "_scales"][pages].to(dtype)[..., None]
        x = x.movedim(-3, -4)
    else:
        x = x.movedim(-2, -4)
    return x.flatten(-3, -2).contiguous()


def _plain_attend(state):
    case = state["case"]
    heads, group, d, prefix = case["heads"], case["group"], case["d"], case["prefix"]
    q = state["q"] * (1 / math.sqrt(d))
    rows, seqs, new = q.shape[0], case["seqs"], case["new"]
    seq, nth, _, real = _places(state, rows)
    starts, lengths = state["starts"].long(), state["lengths"].long()
    counts = starts[1:] - starts[:-1]
    # Each sequence's queries, padded to the most: [seqs, heads, new * group, d].
    index = (starts[:-1, None] + torch.arange(new, device="cuda")).clamp_max(rows - 1)
    padded = q[index].view(seqs, new, heads, group, d).transpose(1, 2).reshape(
        seqs, heads, new * group, d)
    k, v = (_read(state, name, state["pages"].long()) for name in ("k", "v"))
    key = torch.arange(k.shape[-2], device="cuda")
    last = lengths[:, None] - counts[:, None] + torch.arange(new, device="cuda")
    seen = (key <= last[..., None]) & (key < lengths[:, None, None])
    seen = seen[:, None, :, None].expand(-1, 1, -1, group, -1).reshape(seqs, 1, new * group, -1)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous())
    scores = torch.where(seen, scores, -torch.inf)

    def by_row(x):
        x = x.view(seqs, heads, new, group, -1).transpose(1, 2)
        return x[seq, nth.clamp(0, new - 1)]            # [rows, heads, group, ...]

    top = scores.amax(-1, keepdim=True)
    if prefix:
        by_head = q.view(rows, heads, group, d).transpose(0, 1).reshape(heads, rows * group, d)
        pk, pv = (_read(state, name, state["prefix_pages"].long())[:, :prefix].contiguous()
                  for name in ("k", "v"))
        shared = torch.matmul(by_head, pk.transpose(-1, -2).contiguous())
        shared_top = shared.amax(-1, keepdim=True)
        shared = torch.exp(shared - shared_top)
        shared_sum = shared.sum(-1, keepdim=True)
        shared_out = torch.matmul(shared, pv)

        def rows_first(x):
            return x.view(heads, rows, group, -1).transpose(0, 1)

    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total, out = by_row(weights.sum(-1, keepdim=True)), by_row(torch.matmul(weights, v))
    if prefix:
        top, shared_top = by_row(top), rows_first(shared_top)
        most = torch.maximum(top, shared_top)
        a, b = torch.exp(top - most), torch.exp(shared_top - most)
        total = a * total + b * rows_first(shared_sum)
        out = a * out + b * rows_first(shared_out)
    out = torch.where(total == 0, 0.0, out / total)
    return torch.where(real[:, None, None], out.reshape(rows, heads * group, d), 0.0)


def _returned(state):
    names = ("k", "v", "k_scales", "v_scales", "q_out")
    return {name: state[name] for name in names if name in state}


# ---- the framework's calls ----------------------------------------------------------------------

_STREAM = None


def _calls(state):
    """The framework's call on the state's tensors, its descriptor filled as a program fills it once
    for each layer."""
    import mensurflow_amd as mf

    global _STREAM
    if _STREAM is None:
        _STREAM = mf.Stream.wrap(torch.cuda.current_stream().cuda_stream)
    stream = _STREAM
    case = state["case"]

    def array(name, dtype="float32"):
        t = state.get(name)
        return None if t is None else mf.DeviceArray.wrap(t.data_ptr(), tuple(t.shape), stream, dtype,
                                                          t.stride())

    if case["kind"] != "attend":
        scaling, amplitude = _scaling(case)
        rotary = mf.rotary(case["rot"], base=BASE, amplitude=amplitude, **scaling,
                           layout=mf.ROTARY_PAIRS if case["interleaved"] else mf.ROTARY_HALVES)
    if case["kind"] == "rope":
        desc = mf.rope_desc(array("x"), rotary, positions=array("positions", "int32"),
                            backward=case["backward"], out=array("out"))
        return lambda: mf.rope_run(stream, desc)
    held = {"f32": "float32", "bf16": "uint16", "e4m3": "uint8"}[case["held"]]
    k, v = array("k", held), array("v", held)
    if case["held"] != "e4m3":       # [pages, page, heads, d] -> [pages, heads, page, d]
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    cache = mf.KvCache(k, v, array("k_scales"), array("v_scales"))
    batch = mf.KvBatch(array("lengths", "int32"), array("pages", "int32"),
                       starts=array("starts", "int32"), prefix=case.get("prefix", 0),
                       prefix_pages=array("prefix_pages", "int32"))
    if case["kind"] == "append":
        desc = mf.kv_append_desc(cache, batch, array("new_k"), array("new_v"), rotary=rotary,
                                 q=array("q"), q_out=array("q_out"))
        return lambda: mf.kv_append_run(stream, desc)
    desc = mf.attention_paged_desc(array("q"), cache, batch, out=array("out"))
    return lambda: mf.attention_paged_run(stream, desc)


def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        state["call"]()
        return _returned(state) if kind == "append" else {"out": state["out"]}
    if kind == "rope":
        case = state["case"]
        return {"out": _turned(case, state["x"], state["positions"], case["backward"])}
    if kind == "append":
        _plain_append(state)
        return _returned(state)
    return {"out": _plain_attend(state)}


# ---- the work, and the results in 64 bits -------------------------------------------------------


def work(case):
    d = case["d"]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 8 * n * d + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    counts = _counts(case)
    rows = sum(n for n, _ in counts)
    row_bytes = d * BYTES[case["held"]] + (4 if case["held"] == "e4m3" else 0)
    if case["kind"] == "append":
        return {"bytes": rows * (2 * case["heads"] * (4 * d + row_bytes) + 8 * case["q_heads"] * d),
                "flops": rows * (3 * case["rot"] * (case["heads"] + case["q_heads"])
                                 + 4 * case["heads"] * d)}
    pairs = sum(max(0, keys - n + i + 1) for n, keys in counts for i in range(n))
    pairs += rows * case["prefix"]
    q_heads = case["heads"] * case["group"]
    keys = sum(keys for _, keys in counts) + case["prefix"]
    return {"bytes": 2 * keys * case["heads"] * row_bytes + 8 * rows * q_heads * d,
            "flops": 4 * pairs * q_heads * d}


def _nearest_e4m3(v):
    """v (64 bits) on the grid of e4m3: 3 bits behind the leading one, least exponent -6, ties to
    even, at most 448."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_turned(case, x, positions, backward):
    """The rotation as a complex product, in 64 bits."""
    rot, x = case["rot"], x.double()
    if rot == 0:
        return x
    pair = torch.arange(rot // 2, device="cuda")
    first, second = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + rot // 2)
    scaling, amplitude = _scaling(case)
    step = torch.exp(-math.log(BASE) * 2 * pair.double() / rot)
    if scaling:
        kept = (scaling["original"] * step / (2 * math.pi) - scaling["slow"]) / (
            scaling["fast"] - scaling["slow"])
        kept = torch.clamp(kept, 0.0, 1.0)
        step = kept * step + (1 - kept) * step / scaling["factor"]
    angle = torch.outer(positions.double(), step) * (-1 if backward else 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(
        torch.full_like(angle, amplitude), angle)[:, None]
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_append(state):
    case = state["case"]
    starts, lengths = state["starts"].tolist(), state["lengths"].tolist()
    table = state["pages"].tolist()
    out = {name: state[name].double() for name in ("k", "v")}
    scales = {name: state[name + "_scales"].double() for name in out if name + "_scales" in state}
    q_out = state["q_out"].double() if "q" in state else None
    for s, length in enumerate(lengths):
        a, b = starts[s], starts[s + 1]
        place = torch.arange(length - (b - a), length, device="cuda")
        at = torch.tensor(table[s], device="cuda")[place // case["page"]]
        off = place % case["page"]
        for name in out:
            x = state["new_" + name][a:b].double()
            if name == "k":
                x = _exact_turned(case, x, place, False)
            if case["held"] == "e4m3":
                scale = torch.maximum(x.abs().amax(-1) / TOP,
                                      torch.tensor(2.0 ** -126, dtype=torch.float64, device="cuda"))
                scales[name][at, :, off] = scale
                out[name][at, :, off] = _nearest_e4m3(x / scale[..., None])
            else:
                out[name][at, off] = x
        if q_out is not None:
            q_out[a:b] = _exact_turned(case, state["q"][a:b], place, False)
    out.update({name + "_scales": x for name, x in scales.items()})
    if q_out is not None:
        out["q_out"] = q_out
    return out


def _exact_attend(state):
    case = state["case"]
    heads, group, d, prefix = case["heads"], case["group"], case["d"], case["prefix"]
    starts, lengths = state["starts"].tolist(), state["lengths"].tolist()
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    front = [_read(state, name, state["prefix_pages"].long(), torch.float64)[:, :prefix]
             for name in ("k", "v")] if prefix else None
    for s, length in enumerate(lengths):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n == 0 or length + prefix == 0:
            continue
        used = -(-length // case["page"])
        k, v = (_read(state, name, state["pages"][s, :used].long(), torch.float64)[:, :length]
                for name in ("k", "v"))
        if prefix:
            k, v = torch.cat((front[0], k), 1), torch.cat((front[1], v), 1)
        q = state["q"][a:b].double().view(n, heads, group, d).permute(1, 2, 0, 3).reshape(
            heads, group * n, d)
        scores = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        unseen = torch.arange(k.shape[1], device="cuda") > (
            prefix + length - n + torch.arange(n, device="cuda"))[:, None]
        scores.view(heads, group, n, -1).masked_fill_(unseen, -torch.inf)
        top = scores.amax(-1, keepdim=True)
        weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
        total = weights.sum(-1, keepdim=True)
        o = torch.bmm(weights, v) / torch.where(total == 0, 1.0, total)
        out[a:b] = o.view(heads, group, n, d).permute(2, 0, 1, 3).reshape(n, heads * group, d)
    return {"out": out}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return {"out": _exact_turned(case, state["x"], state["positions"], case["backward"])}
    return _exact_append(state) if case["kind"] == "append" else _exact_attend(state)
