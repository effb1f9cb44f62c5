"""The measured cases of the sparse-attention path over the paged cache.

Four operators, in the order a serving step uses them:

  append     rotate the new tokens' queries and keys, write keys and values
             into their cache slots, refresh the summaries of the blocks that
             the tokens landed in
  summarize  the per-channel minimum and maximum of each block's keys, for a
             cache that was filled by something else
  select     score every block of a context by its summary and list the best
  attend     one-token attention over the listed blocks

`run` computes an operator in elementary torch operations, or through libqvp
where `own` is true; `exact` says what it should give in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode step of a 64-sequence batch, 7B-shaped heads, three rotary axes: latency
        dict(name="append 64 tokens", op="append", dtype="bf16", hq=28, hkv=4, dim=128, block=16, layers=1, layer=0,
             batch=64, ctx_lo=1, ctx_hi=512, new_lo=1, new_hi=1, rotary=128, axes=3, interleaved=False, fused=True,
             summary=True, lens_seed=1),
        # prompts of 2,048 tokens out of one fused projection, second chunk of some: bandwidth
        dict(name="append 16 prompts", op="append", dtype="bf16", hq=28, hkv=4, dim=128, block=16, layers=1, layer=0,
             batch=16, ctx_lo=2048, ctx_hi=2300, new_lo=2048, new_hi=2048, rotary=128, axes=3, interleaved=False,
             fused=True, summary=True, lens_seed=2),
        # fp32 cache, neighbouring pairs, half of each head rotated, ragged chunks, one layer of two
        dict(name="append ragged f32", op="append", dtype="f32", hq=8, hkv=2, dim=64, block=16, layers=2, layer=1,
             batch=7, ctx_lo=703, ctx_hi=1501, new_lo=1, new_hi=703, rotary=32, axes=1, interleaved=True, fused=False,
             summary=True, lens_seed=3),
        # summaries of a small fp32 cache: latency
        dict(name="summarize 4 f32", op="summarize", dtype="f32", hq=8, hkv=2, dim=64, block=16, layers=1, layer=0,
             batch=4, ctx_lo=37, ctx_hi=512, lens_seed=4),
        # a serving batch swapped in without summaries
        dict(name="summarize 64 contexts", op="summarize", dtype="bf16", hq=28, hkv=4, dim=128, block=16, layers=1,
             layer=0, batch=64, ctx_lo=512, ctx_hi=8192, lens_seed=5),
        # one long context, 72B-shaped heads: latency
        dict(name="select 1 of 32768", op="select", dtype="bf16", hq=64, hkv=8, dim=128, block=16, layers=1, layer=0,
             batch=1, ctx_lo=32768, ctx_hi=32768, keep=128, sink=1, recent=2, lens_seed=6),
        # an ordinary serving batch, contexts of all lengths
        dict(name="select 64 ragged", op="select", dtype="bf16", hq=28, hkv=4, dim=128, block=16, layers=1, layer=0,
             batch=64, ctx_lo=512, ctx_hi=8192, keep=64, sink=1, recent=2, lens_seed=7),
        # the largest: 32 long contexts
        dict(name="select 32 of 32768", op="select", dtype="bf16", hq=64, hkv=8, dim=128, block=16, layers=1, layer=0,
             batch=32, ctx_lo=32768, ctx_hi=32768, keep=128, sink=1, recent=2, lens_seed=8),
        # attention over the lists of one long context: latency
        dict(name="attend 1 of 32768", op="attend", dtype="bf16", hq=64, hkv=8, dim=128, block=16, layers=1, layer=0,
             batch=1, ctx_lo=32768, ctx_hi=32768, keep=128, sink=1, recent=2, lens_seed=9),
        # an ordinary serving batch; the shortest contexts have fewer blocks than the lists have room for
        dict(name="attend 64 ragged", op="attend", dtype="bf16", hq=28, hkv=4, dim=128, block=16, layers=1, layer=0,
             batch=64, ctx_lo=512, ctx_hi=8192, keep=64, sink=1, recent=2, lens_seed=10),
        # fp32 cache
        dict(name="attend 9 f32", op="attend", dtype="f32", hq=8, hkv=2, dim=64, block=16, layers=2, layer=1,
             batch=9, ctx_lo=37, ctx_hi=2001, keep=33, sink=1, recent=1, lens_seed=11),
        # the largest: 32 long contexts
        dict(name="attend 32 of 32768", op="attend", dtype="bf16", hq=64, hkv=8, dim=128, block=16, layers=1, layer=0,
             batch=32, ctx_lo=32768, ctx_hi=32768, keep=128, sink=1, recent=2, lens_seed=12),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "summarize", "select", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    dim = rng.choice([64, 96, 128, 128])
    block = rng.choice([16, 16, 16, 8, 32])
    layers = rng.choice([1, 1, 2, 3])
    case = dict(op=op, dtype=dtype, hq=hkv * group, hkv=hkv, dim=dim, block=block, layers=layers,
                layer=rng.randrange(layers), lens_seed=rng.randrange(1 << 20))
    if op == "append":
        new = _spread(rng, 1, 2048)
        batch = _spread(rng, 1, max(1, min(64, 16384 // new)))
        axes = rng.choice([1, 3])
        case.update(batch=batch, ctx_lo=new, ctx_hi=new + rng.randrange(300), new_lo=rng.randint(1, new), new_hi=new,
                    rotary=rng.choice([dim, dim, dim // 2]), axes=axes, interleaved=rng.random() < 0.3,
                    fused=rng.random() < 0.5, summary=rng.random() < 0.8)
        return case
    # tokens of the whole cache, all layers: at most about a gigabyte of it
    room = (1 << 29) // (hkv * dim * layers * 2)
    ctx = _spread(rng, 1 if op == "summarize" else 512, min(32768, room))
    batch = _spread(rng, 1, max(1, min(64, room // ctx)))
    case.update(batch=batch, ctx_lo=rng.randint(1, ctx), ctx_hi=ctx)
    if op != "summarize":
        keep = _spread(rng, 4, 160)
        case.update(keep=keep, sink=rng.randrange(3), recent=rng.randrange(3))
    return case


def _lens(case):
    """Context lengths and new tokens of each sequence: part of the case."""
    rng = np.random.default_rng(case["lens_seed"])
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["batch"])
    new = rng.integers(case["new_lo"], case["new_hi"] + 1, size=case["batch"]) if case["op"] == "append" else ctx
    return ctx, np.minimum(new, ctx)


def _elem(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    ctx, new = _lens(case)
    hq, hkv, dim, T, e = case["hq"], case["hkv"], case["dim"], case["block"], _elem(case)
    blocks = -(-ctx // T)
    if case["op"] == "append":
        tokens = int(new.sum())
        touched = int((blocks - (ctx - new) // T).sum())
        moved = tokens * (hq + 2 * hkv) * dim * e * 2 + tokens * case["axes"] * 4
        if case["summary"]:
            moved += touched * hkv * 2 * dim * e
        return {"bytes": moved, "flops": tokens * (hq + hkv) * case["rotary"] * 3}
    if case["op"] == "summarize":
        tokens = int(ctx.sum())
        return {"bytes": tokens * hkv * dim * e + int(blocks.sum()) * hkv * 2 * dim * e, "flops": tokens * hkv * dim * 2}
    q = case["batch"] * hq * dim * e
    listed_bytes = case["batch"] * hkv * case["keep"] * 4
    if case["op"] == "select":
        # a context with no more blocks than the list has room for needs no score
        scored = int((blocks * (blocks > case["keep"])).sum())
        return {"bytes": scored * (hkv * 2 * dim * e + 4) + q + listed_bytes, "flops": scored * hkv * dim * 4}
    tokens = int(np.where(blocks <= case["keep"], ctx, case["keep"] * T).sum())
    return {"bytes": tokens * hkv * dim * e * 2 + 2 * q + listed_bytes, "flops": tokens * hq * dim * 4}


# --- inputs --------------------------------------------------------------------


def _tables(g, blocks):
    """Scattered block ids of every sequence, -1 past its end; pool size."""
    n, pitch = int(blocks.sum()), int(blocks.max())
    total = n + n // 8 + 1
    ids = torch.randperm(total, generator=g, device=DEVICE)[:n].to(torch.int32)
    mapped = torch.arange(pitch, device=DEVICE)[None, :] < torch.as_tensor(blocks, device=DEVICE)[:, None]
    tables = torch.full((len(blocks), pitch), -1, dtype=torch.int32, device=DEVICE)
    tables[mapped] = ids
    return tables, total


def _pool_stride(case):
    n = case["block"] * case["layers"] * case["hkv"] * case["dim"] * 2
    return n, -(-n * _elem(case) // 256) * 256 // _elem(case)


def _summary_stride(case):
    n = case["layers"] * case["hkv"] * case["dim"] * 2
    return n, -(-n * _elem(case) // 256) * 256 // _elem(case)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    ctx, new = _lens(case)
    hq, hkv, dim, T = case["hq"], case["hkv"], case["dim"], case["block"]
    B = case["batch"]
    i32 = dict(dtype=torch.int32, device=DEVICE)
    tables, blocks = _tables(g, -(-ctx // T))
    s = dict(case=case, tables=tables, num_blocks=blocks, ctx=torch.tensor(ctx, **i32), error=torch.zeros(1, **i32),
             max_ctx=int(ctx.max()))
    # keys have channels with an offset and channels of larger spread, as projections give
    offset = torch.randn(hkv, dim, generator=g, device=DEVICE)
    spread = 0.5 + torch.rand(hkv, dim, generator=g, device=DEVICE)

    if case["op"] != "select":
        n, stride = _pool_stride(case)
        s["pool"] = torch.randn(blocks, stride, generator=g, device=DEVICE, dtype=dt)
        view = _pool_view(s)
        view[:, :, 0] *= spread.to(dt)
        view[:, :, 0] += offset.to(dt)
    if case["op"] in ("append", "summarize", "select"):
        n, stride = _summary_stride(case)
        s["summary"] = torch.zeros(blocks, stride, device=DEVICE, dtype=dt)
    if case["op"] == "append":
        most = int(new.max())
        s["new"] = torch.tensor(new, **i32)
        rows = [hq, hkv, hkv]
        if case["fused"]:  # q, k and v of a token side by side, as one projection writes them
            qkv = torch.randn(B, most, sum(rows), dim, generator=g, device=DEVICE, dtype=dt)
            s["q"], s["k"], s["v"] = qkv.split(rows, dim=2)
        else:
            s["q"], s["k"], s["v"] = (torch.randn(B, most, r, dim, generator=g, device=DEVICE, dtype=dt) for r in rows)
        s["q_out"] = torch.zeros(B, most, hq, dim, device=DEVICE, dtype=dt)
        half = case["rotary"] // 2
        s["inv_freq"] = (1e6 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)).float()
        # positions of the new tokens; with three axes, images make them differ from each other and from the slots
        first = torch.tensor(ctx - new, device=DEVICE)
        pos = first[:, None] + torch.arange(most, device=DEVICE)
        shift = torch.randint(0, 64, (case["axes"], B, most), generator=g, device=DEVICE)
        s["pos"] = (pos[None] + (shift if case["axes"] > 1 else 0)).to(torch.int32)
        quarter = half // 4
        s["sections"] = [half] if case["axes"] == 1 else [quarter, (half - quarter) // 2, half - quarter - (half - quarter) // 2]
    elif case["op"] == "select":
        view = _summary_view(s)
        middle = torch.randn(view.shape[:3] + (dim,), generator=g, device=DEVICE) * 0.5 * spread + offset
        reach = (1.2 + 0.6 * torch.rand(middle.shape, generator=g, device=DEVICE)) * spread
        view[:, :, :, 0], view[:, :, :, 1] = (middle - reach).to(dt), (middle + reach).to(dt)
        s["selected"] = torch.zeros(B, hkv, case["keep"], **i32)
    elif case["op"] == "attend":
        nblk = torch.tensor(-(-ctx // T), device=DEVICE)
        score = torch.rand(B, hkv, tables.shape[1], generator=g, device=DEVICE)
        s["selected"] = _lists(score, nblk, case)
        s["out"] = torch.zeros(B, hq, dim, device=DEVICE, dtype=dt)
    if case["op"] in ("select", "attend"):
        s["q"] = torch.randn(B, hq, dim, generator=g, device=DEVICE, dtype=dt)
    return s


def _pool_view(s):
    """[block][layer][K|V][token][kv head][dim] over the pool's bytes."""
    c = s["case"]
    n, _ = _pool_stride(c)
    return s["pool"][:, :n].unflatten(1, (c["layers"], 2, c["block"], c["hkv"], c["dim"]))


def _summary_view(s):
    """[block][layer][kv head][min|max][dim] over the summaries' bytes."""
    c = s["case"]
    n, _ = _summary_stride(c)
    return s["summary"][:, :n].unflatten(1, (c["layers"], c["hkv"], 2, c["dim"]))


def _lists(score, nblk, case):
    """Ascending block numbers of the best scores, -1 past the last: the first
    `sink` and the last `recent` blocks always, ties to the lowest number."""
    keep = case["keep"]
    at = torch.arange(score.shape[-1], device=score.device)
    n = nblk[:, None, None]
    forced = (at < case["sink"]) | (at >= n - case["recent"])
    score = score.masked_fill(forced, math.inf).masked_fill(at >= n, -math.inf)
    ids = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    ids = ids.masked_fill(ids >= n, 1 << 30).sort(dim=-1).values
    out = torch.full(score.shape[:2] + (keep,), -1, dtype=torch.int32, device=score.device)
    out[..., :ids.shape[-1]] = ids.masked_fill(ids == 1 << 30, -1).to(torch.int32)
    return out


# --- the plain forms -------------------------------------------------------------


def run(s):
    return {"append": _append, "summarize": _summarize, "select": _select, "attend": _attend}[s["case"]["op"]](s)


def _rotate(x, cos, sin, rotary, interleaved):
    turned, rest = x[..., :rotary].float(), x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned.chunk(2, dim=-1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _append(s):
    c = s["case"]
    if own:
        return _own_append(s)
    T, most = c["block"], s["k"].shape[1]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEVICE), torch.tensor(s["sections"], device=DEVICE))
    # far positions times a frequency need 64 bits before the circle is closed
    angle = s["pos"].double()[axis].movedim(0, -1) * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    t = torch.arange(most, device=DEVICE)
    live = t < s["new"][:, None]
    s["q_out"][live] = _rotate(s["q"], cos, sin, c["rotary"], c["interleaved"])[live]
    b, t = live.nonzero(as_tuple=True)
    at = (s["ctx"] - s["new"])[b] + t
    ids = s["tables"][b, at // T].long()
    view = _pool_view(s)
    view[ids, c["layer"], 0, at % T] = _rotate(s["k"], cos, sin, c["rotary"], c["interleaved"])[live]
    view[ids, c["layer"], 1, at % T] = s["v"][live]
    if c["summary"]:
        _fill_summaries(s, (s["ctx"] - s["new"]) // T)
    return {"query": s["q_out"], "pool": s["pool"], "summary": s["summary"]}


def _fill_summaries(s, first):
    """Minimum and maximum of the filled slots of blocks first[b], first[b] + 1, ... of every sequence."""
    c = s["case"]
    T = c["block"]
    at = torch.arange(s["tables"].shape[1], device=DEVICE)
    b, j = ((at >= first[:, None]) & (at * T < s["ctx"][:, None])).nonzero(as_tuple=True)
    ids = s["tables"][b, j].long()
    keys = _pool_view(s)[ids, c["layer"], 0].float()
    empty = (torch.arange(T, device=DEVICE) >= (s["ctx"][b] - j * T)[:, None])[:, :, None, None]
    view = _summary_view(s)
    view[ids, c["layer"], :, 0] = keys.masked_fill(empty, math.inf).amin(1).to(view.dtype)
    view[ids, c["layer"], :, 1] = keys.masked_fill(empty, -math.inf).amax(1).to(view.dtype)


def _summarize(s):
    if own:
        return _own_summarize(s)
    _fill_summaries(s, torch.zeros_like(s["ctx"]))
    return s["summary"]


def _select(s):
    c = s["case"]
    if own:
        return _own_select(s)
    q = s["q"].unflatten(1, (c["hkv"], c["hq"] // c["hkv"])).double()  # 64 bits: the choice lies between near values
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    rows = _summary_view(s)[s["tables"].clamp(min=0).long(), c["layer"]].double()
    score = (rows[:, :, :, 1] * up[:, None] + rows[:, :, :, 0] * down[:, None]).sum(-1).movedim(1, 2)
    return _lists(score, (s["ctx"] + c["block"] - 1) // c["block"], c)


def _attend(s):
    c = s["case"]
    if own:
        return _own_attend(s)
    T, B, hkv = c["block"], c["batch"], c["hkv"]
    lists = s["selected"]
    ids = s["tables"].gather(1, lists.clamp(min=0).flatten(1).long()).view_as(lists).long().clamp(min=0)
    kv = _pool_view(s)[ids, c["layer"], :, :, torch.arange(hkv, device=DEVICE)[None, :, None]].float()
    keys, values = kv[:, :, :, 0].flatten(2, 3), kv[:, :, :, 1].flatten(2, 3)
    slot = lists[..., None] * T + torch.arange(T, device=DEVICE)
    hidden = ((lists[..., None] < 0) | (slot >= s["ctx"][:, None, None, None])).flatten(2)
    q = s["q"].unflatten(1, (hkv, -1)).float()
    score = (q @ keys.transpose(2, 3)) * c["dim"] ** -0.5
    score = score.masked_fill(hidden[:, :, None], -math.inf)
    weight = (score - score.amax(-1, keepdim=True)).exp()
    out = (weight @ values.masked_fill(hidden[..., None], 0)) / weight.sum(-1, keepdim=True)
    return out.flatten(1, 2).to(s["q"].dtype)


# --- the framework's calls ---------------------------------------------------------


def _qvp():
    if "qvp" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "qwenvl-paged_b200"))
    import qvp
    return qvp


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _shared(qvp, s):
    """What every call says about the cache."""
    c = s["case"]
    return dict(shape=qvp.make_shape(c["block"], c["layers"], c["hkv"], c["dim"], _elem(c)),
                dtype=qvp.DTYPE_F32 if c["dtype"] == "f32" else qvp.DTYPE_BF16, layer=c["layer"],
                num_blocks=s["num_blocks"], batch=c["batch"], max_blocks_per_seq=s["tables"].shape[1],
                block_tables=s["tables"].data_ptr(), context_lens=s["ctx"].data_ptr(),
                error_word=s["error"].data_ptr())


def _pool_at(s):
    return dict(pool=s["pool"].data_ptr(), block_stride=s["pool"].stride(0) * s["pool"].element_size())


def _summary_at(s):
    return dict(summary=s["summary"].data_ptr(), summary_stride=s["summary"].stride(0) * s["summary"].element_size())


def _own_append(s):
    qvp, c = _qvp(), s["case"]
    if "args" not in s:  # the argument block of a program's buffers, kept as long as they are
        s["args"] = qvp.rope_append_args(
            **_shared(qvp, s), **_pool_at(s), **(_summary_at(s) if c["summary"] else {}), num_query_heads=c["hq"],
            max_query_len=s["q"].shape[1], query_lens=s["new"].data_ptr(), query=s["q"].data_ptr(),
            key=s["k"].data_ptr(), value=s["v"].data_ptr(), query_out=s["q_out"].data_ptr(),
            query_pitch=s["q"].stride(1), key_pitch=s["k"].stride(1), value_pitch=s["v"].stride(1),
            rotary_dim=c["rotary"], rotary_interleaved=int(c["interleaved"]), inv_freq=s["inv_freq"].data_ptr(),
            rope_positions=s["pos"].data_ptr(), rope_sections=s["sections"])
    qvp.check(qvp.rope_append(s["args"], _stream()), "qvp_rope_append")
    return {"query": s["q_out"], "pool": s["pool"], "summary": s["summary"]}


def _own_summarize(s):
    qvp = _qvp()
    if "args" not in s:
        s["args"] = qvp.summarize_args(**_shared(qvp, s), **_pool_at(s), **_summary_at(s), max_context_len=s["max_ctx"])
    qvp.check(qvp.summarize_blocks(s["args"], _stream()), "qvp_summarize_blocks")
    return s["summary"]


def _own_select(s):
    qvp, c = _qvp(), s["case"]
    if "args" not in s:
        s["args"] = qvp.select_args(**_shared(qvp, s), **_summary_at(s), num_query_heads=c["hq"],
                                    max_context_len=s["max_ctx"], query=s["q"].data_ptr(), max_selected=c["keep"],
                                    sink_blocks=c["sink"], recent_blocks=c["recent"], selected=s["selected"].data_ptr())
    qvp.check(qvp.select_blocks(s["args"], _stream()), "qvp_select_blocks")
    return s["selected"]


def _own_attend(s):
    qvp, c = _qvp(), s["case"]
    if "args" not in s:
        s["args"] = qvp.decode_selected_args(**_shared(qvp, s), **_pool_at(s), num_query_heads=c["hq"],
                                             scale=c["dim"] ** -0.5, query=s["q"].data_ptr(),
                                             selected=s["selected"].data_ptr(), max_selected=c["keep"],
                                             out=s["out"].data_ptr())
    qvp.check(qvp.decode_selected(s["args"], _stream()), "qvp_decode_selected")
    return s["out"]


# --- what they should give, in 64 bits --------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "summarize": _exact_summarize, "select": _exact_select,
            "attend": _exact_attend}[case["op"]](case, s)


def _exact_append(c, s):
    T, L, half = c["block"], c["layer"], c["rotary"] // 2
    pool, query, summary = (s[k].double() for k in ("pool", "q_out", "summary"))
    slots = pool[:, :_pool_stride(c)[0]].unflatten(1, (c["layers"], 2, T, c["hkv"], c["dim"]))
    bounds = summary[:, :_summary_stride(c)[0]].unflatten(1, (c["layers"], c["hkv"], 2, c["dim"]))
    ends = np.cumsum(s["sections"])
    ctx, new = _lens(c)
    for b in range(c["batch"]):
        n, start = int(new[b]), int(ctx[b] - new[b])
        turn = torch.empty(n, half, dtype=torch.complex128, device=DEVICE)
        for x, end in enumerate(ends):
            lo = int(ends[x - 1]) if x else 0
            a = torch.outer(s["pos"][x, b, :n].double(), s["inv_freq"][lo:int(end)].double())
            turn[:, lo:int(end)] = torch.polar(torch.ones_like(a), a)

        def turned(rows):
            rows = rows[b, :n].double().clone()
            head = rows[..., :c["rotary"]]
            first, second = (head[..., 0::2], head[..., 1::2]) if c["interleaved"] else (head[..., :half], head[..., half:])
            z = torch.complex(first.contiguous(), second.contiguous()) * turn[:, None]
            first.copy_(z.real), second.copy_(z.imag)
            return rows

        query[b, :n] = turned(s["q"])
        at = torch.arange(start, start + n, device=DEVICE)
        frames = s["tables"][b].long()[at // T]
        slots[frames, L, 0, at % T] = turned(s["k"])
        slots[frames, L, 1, at % T] = s["v"][b, :n].double()
        if c["summary"]:
            blocks = range(start // T, -(-int(ctx[b]) // T))
            whole = s["tables"][b, blocks.start:blocks.stop].long()
            filled = slots[whole, L, 0]
            last = int(ctx[b]) - (blocks.stop - 1) * T
            bounds[whole, L, :, 0], bounds[whole, L, :, 1] = filled.amin(1), filled.amax(1)
            bounds[whole[-1], L, :, 0] = filled[-1, :last].amin(0)
            bounds[whole[-1], L, :, 1] = filled[-1, :last].amax(0)
    return {"query": query, "pool": pool, "summary": summary}


def _exact_summarize(c, s):
    T, ctx = c["block"], _lens(c)[0]
    pool = s["pool"][:, :_pool_stride(c)[0]].unflatten(1, (c["layers"], 2, T, c["hkv"], c["dim"]))
    out = s["summary"].double()
    bounds = out[:, :_summary_stride(c)[0]].unflatten(1, (c["layers"], c["hkv"], 2, c["dim"]))
    for b in range(c["batch"]):
        n = int(ctx[b])
        frames = s["tables"][b, :-(-n // T)].long()
        rows = pool[frames, c["layer"], 0].double()
        bounds[frames, c["layer"], :, 0], bounds[frames, c["layer"], :, 1] = rows.amin(1), rows.amax(1)
        rest = n - (len(frames) - 1) * T
        bounds[frames[-1], c["layer"], :, 0] = rows[-1, :rest].amin(0)
        bounds[frames[-1], c["layer"], :, 1] = rows[-1, :rest].amax(0)
    return out


def _exact_select(c, s):
    G, T, keep, ctx = c["hq"] // c["hkv"], c["block"], c["keep"], _lens(c)[0]
    bounds = s["summary"][:, :_summary_stride(c)[0]].unflatten(1, (c["layers"], c["hkv"], 2, c["dim"]))
    out = torch.full((c["batch"], c["hkv"], keep), -1, dtype=torch.int32)
    for b in range(c["batch"]):
        n = -(-int(ctx[b]) // T)
        rows = bounds[s["tables"][b, :n].long(), c["layer"]].double()
        for h in range(c["hkv"]):
            q = s["q"][b, h * G:(h + 1) * G].double()
            # the largest product that a key inside the bounds can reach, channel by channel
            reach = torch.maximum(q[:, None] * rows[None, :, h, 0], q[:, None] * rows[None, :, h, 1]).sum((0, 2)).tolist()
            if n <= keep:
                chosen = list(range(n))
            else:
                always = set(range(c["sink"])) | set(range(n - c["recent"], n))
                rest = sorted((j for j in range(n) if j not in always), key=lambda j: (-reach[j], j))
                chosen = sorted(always) + rest[:keep - len(always)]
            out[b, h, :len(chosen)] = torch.tensor(sorted(chosen), dtype=torch.int32)
    return out


def _exact_attend(c, s):
    G, T, ctx = c["hq"] // c["hkv"], c["block"], _lens(c)[0]
    pool = s["pool"][:, :_pool_stride(c)[0]].unflatten(1, (c["layers"], 2, T, c["hkv"], c["dim"]))
    out = torch.empty(c["batch"], c["hq"], c["dim"], dtype=torch.float64, device=DEVICE)
    lists = s["selected"].tolist()
    for b in range(c["batch"]):
        for h in range(c["hkv"]):
            chosen = torch.tensor([j for j in lists[b][h] if j >= 0], device=DEVICE)
            rows = pool[s["tables"][b].long()[chosen], c["layer"], :, :, h].double()
            at = (chosen[:, None] * T + torch.arange(T, device=DEVICE)).flatten()
            seen = at < int(ctx[b])
            keys, values = rows[:, 0].flatten(0, 1)[seen], rows[:, 1].flatten(0, 1)[seen]
            q = s["q"][b, h * G:(h + 1) * G].double()
            out[b, h * G:(h + 1) * G] = torch.softmax(q @ keys.T / math.sqrt(c["dim"]), dim=-1) @ values
    return out
