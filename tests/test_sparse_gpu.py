"""The sparse-attention calls on the GPU against their definitions in 64 bits.

Tolerances. A result rounded to the element type is off by at most half a step
of it: 2^-8 of the value in bf16, 2^-24 in fp32 (STEP). To that comes:

* a rotated element x cos a - y sin a, in 32 bits: the angle's remainder is
  rounded at 2^-25 of half a turn (pi 2^-25), the cosine and sine at 2^-23
  (twice the bound of one ulp), two products and a sum at 2^-24 each, all in
  proportion to |x| + |y|: less than 2^-21 (|x| + |y|);
* attention: a score s = scale <q, k> summed in 32 bits is off by at most
  (D + 4) 2^-23 of scale sum_d |q_d k_d| <= reach, which moves a weight by that
  factor; the power of two, the sum of N weights and the final product add
  2^-21 + N 2^-24. Numerator and denominator are both off by it, so out is off
  by 2 (...) sum_t p_t |v_t|. Where the weights are multiplied as two bf16
  terms, they lose 2^-16; as one bf16, 2^-8.
"""
import ctypes as C
import importlib.util
import itertools
import math
import os
import random

import numpy as np
import pytest

import qvp
import sparse_oracle as S

pytestmark = pytest.mark.gpu

STEP = {"bf16": 2.0**-8, "f32": 2.0**-24}


def _torch():
    import torch
    return torch


def _dtype(name):
    torch = _torch()
    return torch.bfloat16 if name == "bf16" else torch.float32


def _stream():
    return _torch().cuda.current_stream().cuda_stream


class Cache:
    """A cache with scattered tables on cuda:0, its summaries, and 64-bit copies of both."""

    def __init__(self, seed, ctx, *, dtype="bf16", layers=1, layer=0, T=16, hkv=2, D=64, pitch=None, pad=0,
                 offset=0, fill=1.0, spare=3):
        torch = _torch()
        self.dtype, self.layer, self.T, self.hkv, self.D, self.layers = dtype, layer, T, hkv, D, layers
        self.ctx = np.asarray(ctx, dtype=np.int32)
        self.rng = np.random.default_rng(seed)
        need = -(-self.ctx // T)
        self.pitch = pitch or max(1, int(need.max()))
        self.blocks = int(need.sum()) + spare
        ids = self.rng.permutation(self.blocks)
        self.tables = np.full((len(ctx), self.pitch), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = ids[at:at + n]
            at += n
        self.shape = qvp.make_shape(T, layers, hkv, D, 2 if dtype == "bf16" else 4)
        elem = self.shape.bytes_per_element
        self.stride = qvp.block_stride(self.shape) // elem + pad
        self.sum_stride = qvp.block_stride(qvp.summary_shape(self.shape)) // elem + pad
        self.n = T * layers * hkv * D * 2
        self.sum_n = layers * hkv * D * 2
        self.pool = self.make((self.blocks, self.stride), offset, fill)
        self.summary = self.make((self.blocks, self.sum_stride), offset, fill)
        self.tables_d = torch.from_numpy(self.tables).cuda()
        self.ctx_d = torch.from_numpy(self.ctx).cuda()
        self.error = torch.zeros(1, dtype=torch.int32, device="cuda")

    def make(self, shape, offset=0, scale=1.0):
        """Normal values in the element type, `offset` elements past an aligned address."""
        torch = _torch()
        x = self.rng.standard_normal(math.prod(shape) + offset, dtype=np.float32) * scale
        return torch.from_numpy(x).to(_dtype(self.dtype)).cuda()[offset:].view(shape)

    def pool64(self):
        x = self.pool.double().cpu().numpy()[:, :self.n]
        return x.reshape(self.blocks, self.layers, 2, self.T, self.hkv, self.D)

    def summary64(self):
        x = self.summary.double().cpu().numpy()[:, :self.sum_n]
        return x.reshape(self.blocks, self.layers, self.hkv, 2, self.D)

    def common(self, **kw):
        base = dict(shape=self.shape, dtype=qvp.DTYPE_BF16 if self.dtype == "bf16" else qvp.DTYPE_F32,
                    layer=self.layer, num_blocks=self.blocks, batch=len(self.ctx), max_blocks_per_seq=self.pitch,
                    block_tables=self.tables_d.data_ptr(), context_lens=self.ctx_d.data_ptr(),
                    error_word=self.error.data_ptr())
        base.update(kw)
        return base

    def at_pool(self):
        return dict(pool=self.pool.data_ptr(), block_stride=self.stride * self.shape.bytes_per_element)

    def at_summary(self):
        return dict(summary=self.summary.data_ptr(), summary_stride=self.sum_stride * self.shape.bytes_per_element)

    def summarize(self, **kw):
        args = qvp.summarize_args(**self.common(max_context_len=max(1, int(self.ctx.max())), **self.at_pool(),
                                                **self.at_summary(), **kw))
        assert qvp.summarize_blocks(args, _stream()) == qvp.OK, qvp.last_error()

    def select_args(self, q, keep, sink, recent, **kw):
        torch = _torch()
        out = torch.full((len(self.ctx), self.hkv, keep), -7, dtype=torch.int32, device="cuda")
        base = self.common(num_query_heads=q.shape[1], max_context_len=max(1, int(self.ctx.max())),
                           query=q.data_ptr(), query_pitch=q.stride(0), max_selected=keep, sink_blocks=sink,
                           recent_blocks=recent, selected=out.data_ptr(), **self.at_summary())
        base.update(kw)
        return qvp.select_args(**base), out

    def attend_args(self, q, selected, scale=None, **kw):
        torch = _torch()
        out = torch.full((len(self.ctx), q.shape[1], self.D), -7.0, dtype=_dtype(self.dtype), device="cuda")
        base = self.common(num_query_heads=q.shape[1], scale=scale or self.D ** -0.5, query=q.data_ptr(),
                           query_pitch=q.stride(0), selected=selected.data_ptr(), max_selected=selected.shape[2],
                           out=out.data_ptr(), **self.at_pool())
        base.update(kw)
        return qvp.decode_selected_args(**base), out

    def errors(self):
        _torch().cuda.synchronize()
        return int(self.error.item())


def _bits(x):
    torch = _torch()
    return x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.int32).cpu().numpy().copy()


# --- rotary append -------------------------------------------------------------


def run_append(c, new, hq, *, most=None, rotary=None, sections=None, interleaved=False, positions="random",
               fused=False, in_place=False, summary=True, offset=0, extra_pitch=0, inv_freq=None):
    """Appends random q, k, v and checks every byte of the outputs and of what must not change."""
    torch = _torch()
    new = np.asarray(new, dtype=np.int32)
    B, most = len(new), most or max(1, int(new.max()))
    D, hkv, T = c.D, c.hkv, c.T
    rotary = D if rotary is None else rotary
    half = rotary // 2
    sections = sections or [half]
    rows = [hq, hkv, hkv]
    if fused:
        qkv = c.make((B, most, sum(rows), D), offset)
        q, k, v = qkv.split(rows, dim=2)
    else:
        q, k, v = (c.make((B, most, r * D + extra_pitch), offset)[..., :r * D].unflatten(-1, (r, D)) for r in rows)
    q64, k64, v64 = (x.double().cpu().numpy() for x in (q, k, v))
    out = q if in_place else c.make((B, most, hq, D), offset)
    out_before, pool_before, summary_before = _bits(out), _bits(c.pool), _bits(c.summary)
    pool64 = c.pool64().copy()
    if inv_freq is None:
        inv_freq = (1e4 ** (-np.arange(half) / max(1, half))).astype(np.float32)
    freq = torch.from_numpy(inv_freq).cuda()
    pos = pos_d = None
    if positions == "random":
        # up to 2^24: there the oracle's own angle is good to 2^-29
        pos = c.rng.integers(0, 2**24, size=(len(sections), B, most)).astype(np.int32)
        pos[:, :, ::2] %= 4096
    elif positions is not None:
        pos = positions
    if pos is not None:
        pos_d = torch.from_numpy(pos).cuda()
    new_d = torch.from_numpy(new).cuda()
    args = qvp.rope_append_args(
        **c.common(), **c.at_pool(), **(c.at_summary() if summary else {}), num_query_heads=hq, max_query_len=most,
        query_lens=new_d.data_ptr(), query=q.data_ptr() if hq else 0, key=k.data_ptr(), value=v.data_ptr(),
        query_out=out.data_ptr() if hq else 0, query_pitch=q.stride(1) if hq else 0, key_pitch=k.stride(1),
        value_pitch=v.stride(1), rotary_dim=rotary, rotary_interleaved=int(interleaved),
        inv_freq=freq.data_ptr() if half else 0, rope_positions=pos_d.data_ptr() if pos is not None else 0,
        rope_sections=sections if pos is not None else [])
    assert qvp.rope_append(args, _stream()) == qvp.OK, qvp.last_error()
    assert c.errors() == 0

    want_q, writes, filled = S.rope_append(pool64, c.tables, c.ctx, new, c.layer, q64, k64, v64, inv_freq, pos,
                                           sections, interleaved)
    live = np.arange(most)[None, :] < new[:, None]

    def near(got, want, x):
        """Rotated elements: both parts of a pair bound each other's error."""
        size = np.abs(x)
        bound = np.zeros_like(size)
        i, j = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if interleaved else \
            (np.arange(half), np.arange(half, rotary))
        bound[..., i] = bound[..., j] = size[..., i] + size[..., j]
        assert (np.abs(got - want) <= STEP[c.dtype] * np.abs(want) + 2.0**-21 * bound).all()

    if hq:
        got = out.double().cpu().numpy()
        near(got[live], want_q[live], q64[live])
        if not in_place:
            assert np.array_equal(_bits(out)[~live], out_before[~live])
    after = c.pool64()
    changed = np.zeros(pool64.shape, dtype=bool)
    for n, (block, slot, krow, vrow) in enumerate(writes):
        changed[block, c.layer, :, slot] = True
    k_by_slot = {}
    for b, t in zip(*live.nonzero()):
        at = int(c.ctx[b]) - int(new[b]) + t
        k_by_slot[(int(c.tables[b, at // T]), at % T)] = k64[b, t]
    for block, slot, krow, vrow in writes:
        near(after[block, c.layer, 0, slot], krow, k_by_slot[(block, slot)])
        assert np.array_equal(after[block, c.layer, 1, slot], vrow)
    kept = np.ones(pool_before.shape, dtype=bool)
    kept[:, :c.n] = ~changed.reshape(c.blocks, -1)
    assert np.array_equal(_bits(c.pool)[kept], pool_before[kept])
    # summaries: of the keys as they are stored, bit for bit
    kept = np.ones(summary_before.shape, dtype=bool)
    if summary:
        got = c.summary64()
        touched = np.zeros((c.blocks, c.layers, c.hkv, 2, D), dtype=bool)
        for block, n in filled.items():
            assert np.array_equal(got[block, c.layer], S.summary_of(after, block, c.layer, n))
            touched[block, c.layer] = True
        kept[:, :c.sum_n] = ~touched.reshape(c.blocks, -1)
    assert np.array_equal(_bits(c.summary)[kept], summary_before[kept])
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,D,T", [(28, 4, 128, 16), (8, 2, 64, 16), (5, 5, 80, 16), (3, 1, 96, 8),
                                        (2, 2, 256, 32), (7, 1, 33, 5), (4, 4, 8, 1), (40, 40, 64, 48)])
def test_append_over_shapes(dtype, hq, hkv, D, T):
    ctx = [1, 17, 16, 45, 33, 70]
    new = [1, 17, 1, 20, 0, 23]
    c = Cache(1, ctx, dtype=dtype, layers=2, layer=1, T=T, hkv=hkv, D=D)
    run_append(c, new, hq, rotary=D // 2 * 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary,sections", [(0, None), (2, [1]), (32, [16]), (64, [8, 12, 12]), (64, [0, 32]),
                                             (48, [24, 0, 0, 0]), (62, [31])])
def test_append_over_rotations(dtype, interleaved, rotary, sections):
    c = Cache(2, [40, 9, 31], dtype=dtype, hkv=2, D=64)
    run_append(c, [11, 9, 1], 6, rotary=rotary, sections=sections, interleaved=interleaved)


def test_append_single_tokens_of_a_batch_with_padding_rows():
    c = Cache(3, [512, 1, 0, 16, 17, 300], hkv=4, D=128, pitch=40)
    run_append(c, [1, 1, 0, 1, 1, 0], 28, sections=[16, 24, 24])


@pytest.mark.parametrize("new", [[0, 0], [700, 1], [33, 700]])
def test_append_long_chunks(new):
    c = Cache(4, [703, 765], hkv=2, D=64)
    run_append(c, new, 4, most=701)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hkv,D", [(8, 128), (5, 64), (7, 80), (40, 64), (3, 33)])
@pytest.mark.parametrize("kw", [dict(), dict(summary=False, fused=True), dict(hq=0)])
def test_append_where_ctas_share_a_blocks_kv_heads(dtype, hkv, D, kw):
    """Few blocks and many kv heads: even and uneven shares, old tokens of a block, an empty chunk."""
    c = Cache(41, [13, 29, 0, 40], dtype=dtype, layers=2, layer=1, hkv=hkv, D=D)
    kw = dict(kw)
    run_append(c, [13, 9, 0, 1], kw.pop("hq", hkv), rotary=D // 4 * 2, **kw)


@pytest.mark.parametrize("dtype,hq,hkv,D,T,most", [("bf16", 16, 4, 64, 8, 200), ("bf16", 17, 1, 64, 16, 400),
                                                   ("f32", 8, 2, 64, 16, 400), ("bf16", 12, 2, 256, 8, 200),
                                                   ("f32", 4, 1, 256, 8, 200), ("bf16", 10, 5, 96, 16, 400)])
@pytest.mark.parametrize("kw", [dict(), dict(fused=True, interleaved=True), dict(in_place=True, rotary=32)])
def test_append_prompts_of_a_full_batch(dtype, hq, hkv, D, T, most, kw):
    """Several waves of CTAs whose threads take several heads each; lengths from none to all rows."""
    rng = np.random.default_rng(37)
    new = rng.integers(0, most + 1, size=24)
    new[:5] = most, 0, 1, most - 1, T
    c = Cache(38, new + rng.integers(0, 3 * T, size=24), dtype=dtype, hkv=hkv, D=D, T=T)
    run_append(c, new, hq, most=most, **kw)


def test_append_cache_positions_are_the_default():
    c = Cache(5, [100, 37], hkv=2, D=64)
    run_append(c, [40, 37], 4, positions=None)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw", [dict(fused=True), dict(extra_pitch=3), dict(offset=1), dict(in_place=True),
                                dict(summary=False)])
def test_append_over_strides_and_alignments(dtype, kw):
    for pad, offset in ((0, 0), (8, 0), (1, 0), (0, 1)):
        c = Cache(6, [50, 20, 31], dtype=dtype, hkv=2, D=64, pad=pad, offset=offset)
        run_append(c, [30, 20, 1], 4, **kw)


def test_append_keys_and_values_alone():
    c = Cache(7, [50, 20], hkv=2, D=64)
    run_append(c, [30, 20], 0)


def test_append_over_earlier_tokens_leaves_no_trace_in_the_summary():
    torch = _torch()
    c = Cache(8, [40], hkv=1, D=64)
    c.pool.mul_(100)  # what was there is far outside the new keys
    run_append(c, [40], 2, sections=[32])
    c.ctx[:] = 36
    c.ctx_d.copy_(torch.from_numpy(c.ctx))
    run_append(c, [3], 2, sections=[32])
    assert np.abs(c.summary64()[c.tables[0]]).max() < 50


def test_append_keeps_nan_and_infinity():
    torch = _torch()
    c = Cache(9, [20], dtype="f32", hkv=1, D=8, T=16)
    k = torch.zeros(1, 20, 1, 8, device="cuda")
    k[0, 3, 0, 1], k[0, 5, 0, 2], k[0, 6, 0, 3] = math.nan, math.inf, -math.inf
    new = torch.tensor([20], dtype=torch.int32, device="cuda")
    args = qvp.rope_append_args(**c.common(), **c.at_pool(), **c.at_summary(), num_query_heads=0, max_query_len=20,
                                query_lens=new.data_ptr(), key=k.data_ptr(), value=k.data_ptr())
    assert qvp.rope_append(args, _stream()) == qvp.OK and c.errors() == 0
    lo, hi = c.summary64()[c.tables[0, 0], 0, 0]
    assert np.isnan([lo[1], hi[1]]).all() and hi[2] == np.inf and lo[2] == 0 and lo[3] == -np.inf and hi[3] == 0
    c.pool.zero_(), c.summary.zero_()
    c.pool.view(c.blocks, -1)[:, :c.n].view(c.blocks, 2, 16, 8)[int(c.tables[0, 0]), 0, :20].copy_(k[0, :16, 0])
    c.summarize()
    again = c.summary64()[c.tables[0, 0], 0, 0]
    assert np.array_equal(again, np.stack((lo, hi)), equal_nan=True)


@pytest.mark.parametrize("change,bit", [
    (dict(ctx=[-1, 20]), 4), (dict(ctx=[65, 20]), 4), (dict(ctx=[3, 20]), 4), (dict(new=[-1, 4]), 4),
    (dict(new=[9, 4]), 4), (dict(table=-1), 1), (dict(table=10**6), 1)])
def test_append_flags_bad_lengths_and_ids_and_serves_the_rest(change, bit):
    torch = _torch()
    c = Cache(10, [40, 20], hkv=1, D=64, pitch=4)
    before = _bits(c.pool)
    ctx = torch.tensor(change.get("ctx", [40, 20]), dtype=torch.int32, device="cuda")
    new = torch.tensor(change.get("new", [4, 4]), dtype=torch.int32, device="cuda")
    if "table" in change:
        c.tables_d[0, 2] = change["table"]
    k, v = c.make((2, 8, 1, 64)), c.make((2, 8, 1, 64))
    args = qvp.rope_append_args(**c.common(context_lens=ctx.data_ptr()), **c.at_pool(), **c.at_summary(),
                                num_query_heads=0, max_query_len=8, query_lens=new.data_ptr(), key=k.data_ptr(),
                                value=v.data_ptr())
    assert qvp.rope_append(args, _stream()) == qvp.OK
    assert c.errors() == bit
    after = _bits(c.pool)
    served = np.zeros(before.shape, dtype=bool)
    block = int(c.tables[1, 1])  # tokens 16 .. 19 of the second sequence, slots 0 .. 3
    served[block].reshape(2, 16, 64)[:, :4] = True
    assert np.array_equal(after[~served], before[~served])
    want = np.stack((_bits(k)[1, :4, 0], _bits(v)[1, :4, 0]))
    assert np.array_equal(after[block].reshape(2, 16, 64)[:, :4], want)


@pytest.mark.parametrize("change,bit", [
    (dict(ctx=[-1, 20]), 4), (dict(ctx=[65, 20]), 4), (dict(ctx=[9, 20]), 4), (dict(new=[-1, 4]), 4),
    (dict(new=[13, 4]), 4), (dict(table=-1), 1), (dict(table=10**6), 1)])
@pytest.mark.parametrize("dtype,hq,hkv", [("bf16", 6, 3), ("f32", 4, 1)])
def test_append_leaves_queries_and_summaries_of_bad_lengths_alone(change, bit, dtype, hq, hkv):
    """A bad length leaves out its sequence; a bad id leaves out its block, whose queries are rotated all the same."""
    torch = _torch()
    c = Cache(40, [40, 20], dtype=dtype, hkv=hkv, D=64, pitch=4)
    q, k, v = (c.make((2, 12, h, 64)) for h in (hq, hkv, hkv))
    freq = torch.from_numpy((1e4 ** (-np.arange(32) / 32)).astype(np.float32)).cuda()
    before = [c.pool.clone(), c.summary.clone(), c.make((2, 12, hq, 64))]

    def append(ctx, new, pool, summary, out):
        ctx, new = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ctx, new))
        c.pool, c.summary = pool, summary
        args = qvp.rope_append_args(**c.common(context_lens=ctx.data_ptr()), **c.at_pool(), **c.at_summary(),
                                    num_query_heads=hq, max_query_len=12, query_lens=new.data_ptr(),
                                    query=q.data_ptr(), key=k.data_ptr(), value=v.data_ptr(),
                                    query_out=out.data_ptr(), rotary_dim=64, inv_freq=freq.data_ptr())
        assert qvp.rope_append(args, _stream()) == qvp.OK
        return c.errors()

    good = [x.clone() for x in before]
    assert append([40, 20], [10, 4], *good) == 0
    if "table" in change:
        c.tables_d[0, 2] = change["table"]
    got = [x.clone() for x in before]
    assert append(change.get("ctx", [40, 20]), change.get("new", [10, 4]), *got) == bit
    served = [int(c.tables[1, 1])]               # tokens 16 .. 19 of the second sequence
    if bit == 1:
        served.append(int(c.tables[0, 1]))       # tokens 30 and 31 of the first: 32 .. 39 have no block
    for i in range(2):
        want = before[i].clone()
        want[served] = good[i][served]
        assert np.array_equal(_bits(got[i]), _bits(want))
    want = good[2].clone()
    if bit == 4:
        want[0] = before[2][0]
    assert np.array_equal(_bits(got[2]), _bits(want))


# --- summaries -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hkv,D,T,pad,offset", [(4, 128, 16, 0, 0), (2, 64, 16, 8, 0), (1, 96, 8, 0, 0),
                                                (3, 33, 5, 0, 0), (2, 64, 16, 1, 0), (2, 64, 16, 0, 1),
                                                (1, 8, 1, 0, 0), (2, 256, 40, 0, 0)])
@pytest.mark.parametrize("first", [None, [0, 0, 18, 40, 37, 1]])
def test_summaries_match_the_definition_bit_for_bit(dtype, hkv, D, T, pad, offset, first):
    torch = _torch()
    ctx = [1, 0, 33, 40, 37, 129]
    c = Cache(11, ctx, dtype=dtype, layers=2, layer=1, T=T, hkv=hkv, D=D, pad=pad, offset=offset)
    before = _bits(c.summary)
    first_d = torch.tensor(first or [0] * 6, dtype=torch.int32, device="cuda")
    c.summarize(first_tokens=first_d.data_ptr() if first else 0)
    assert c.errors() == 0
    got, pool = c.summary64(), c.pool64()
    kept = np.ones((c.blocks, c.layers, hkv, 2, D), dtype=bool)
    for b, n in enumerate(ctx):
        start = first[b] if first else 0
        if start >= n:
            continue
        for j in range(start // T, -(-n // T)):
            block = int(c.tables[b, j])
            assert np.array_equal(got[block, 1], S.summary_of(pool, block, 1, min(T, n - j * T)))
            kept[block, 1] = False
    mask = np.ones(before.shape, dtype=bool)
    mask[:, :c.sum_n] = kept.reshape(c.blocks, -1)
    assert np.array_equal(_bits(c.summary)[mask], before[mask])


@pytest.mark.parametrize("ctx,first,table,bit", [([-1, 20], 0, None, 4), ([49, 20], 0, None, 4), ([40, 20], -1, None, 4),
                                                 ([40, 20], 0, -1, 1), ([40, 20], 0, 999, 1)])
def test_summaries_flag_bad_lengths_and_ids(ctx, first, table, bit):
    torch = _torch()
    c = Cache(12, [40, 20], hkv=1, D=64, pitch=3)
    before, pool = _bits(c.summary), c.pool64()
    ctx_d = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    first_d = torch.tensor([first, 0], dtype=torch.int32, device="cuda")
    if table is not None:
        c.tables_d[0, :] = table
    args = qvp.summarize_args(**c.common(context_lens=ctx_d.data_ptr(), max_context_len=48), **c.at_pool(),
                              **c.at_summary(), first_tokens=first_d.data_ptr())
    assert qvp.summarize_blocks(args, _stream()) == qvp.OK
    assert c.errors() == bit
    good = c.tables[1, :2]
    got = c.summary64()
    for j, block in enumerate(good):
        assert np.array_equal(got[block, 0], S.summary_of(pool, int(block), 0, [16, 4][j]))
    others = np.setdiff1d(np.arange(c.blocks), good)
    assert np.array_equal(_bits(c.summary)[others], before[others])


# --- selection -----------------------------------------------------------------


def run_select(c, q, keep, sink, recent, **kw):
    args, out = c.select_args(q, keep, sink, recent, **kw)
    assert qvp.select_blocks(args, _stream()) == qvp.OK, qvp.last_error()
    assert c.errors() == 0
    want = S.select(q.double().cpu().numpy(), c.summary64(), c.tables, c.ctx, c.T, c.layer, c.hkv, keep, sink, recent)
    assert np.array_equal(out.cpu().numpy(), want)
    return out


def sort_summaries(c):
    """Random summaries whose minimum is below their maximum."""
    torch = _torch()
    v = c.summary[:, :c.sum_n].unflatten(1, (c.layers, c.hkv, 2, c.D))
    lo, hi = torch.minimum(v[..., 0, :], v[..., 1, :]), torch.maximum(v[..., 0, :], v[..., 1, :])
    v[..., 0, :], v[..., 1, :] = lo, hi


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,D,T", [(28, 4, 128, 16), (8, 2, 64, 16), (5, 1, 96, 8), (6, 3, 80, 32),
                                        (2, 2, 256, 16), (7, 1, 33, 5), (4, 1, 16, 1), (16, 1, 128, 16)])
@pytest.mark.parametrize("keep,sink,recent", [(8, 1, 2), (1, 0, 0), (5, 2, 3), (13, 0, 1)])
def test_select_matches_the_definition(dtype, hq, hkv, D, T, keep, sink, recent):
    # from no block to many, and the counts on either side of the list's length
    ctx = [0, 1, keep * T, keep * T + 1, (keep + 1) * T, 90 * T - 1, 200 * T, 63 * T + 2]
    c = Cache(13, ctx, dtype=dtype, layers=2, layer=1, T=T, hkv=hkv, D=D)
    sort_summaries(c)
    run_select(c, c.make((len(ctx), hq, D)), keep, sink, recent)


@pytest.mark.parametrize("blocks,keep", [(2000, 64), (2000, 1999), (2000, 700), (70000, 128), (513, 512)])
@pytest.mark.parametrize("batch", [1, 40])
def test_select_over_long_contexts(blocks, keep, batch):
    if batch > 1 and blocks > 2000:
        pytest.skip("the oracle would take minutes")
    ctx = [blocks * 16 - 3] + [blocks * 8] * (batch - 1)
    c = Cache(14, ctx, hkv=1, D=64, T=16) if blocks <= 2000 else Cache(14, ctx, hkv=1, D=16, T=16)
    sort_summaries(c)
    run_select(c, c.make((batch, 4, c.D)), keep, 1, 0)


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f32", 16)])
@pytest.mark.parametrize("blocks,ctx", [(114688, [114690, 100, 101, 102, 5000, 0]),      # eight CTAs, each full
                                        (14336, [14338] + [90] * 80 + [130, 0] * 40),   # one CTA a context, full
                                        (14337, [14339] + [90] * 80 + [130, 0] * 40)])  # a second one for the last block
def test_select_where_ctas_hold_all_the_blocks_they_can(dtype, D, blocks, ctx):
    c = Cache(39, ctx, dtype=dtype, hkv=1, D=D, T=1)
    sort_summaries(c)
    run_select(c, c.make((len(ctx), 3, D)), 100, 1, 1, max_context_len=blocks + 2)


@pytest.mark.parametrize("kind", ["equal", "two", "few", "steep", "zeros", "outlier", "tiny"])
@pytest.mark.parametrize("batch", [1, 64])
def test_select_where_scores_tie_or_crowd(kind, batch):
    """Equal scores go to the lower block, whatever the distribution does to the search."""
    torch = _torch()
    blocks = 1500 if batch == 1 else 300
    c = Cache(15, [blocks * 16] * batch, dtype="f32", hkv=1, D=64)
    v = c.summary[:, :c.sum_n].view(c.blocks, 2, 64)
    rng = np.random.default_rng(16)
    x = {"equal": np.ones(c.blocks), "two": rng.integers(0, 2, c.blocks), "few": rng.integers(0, 5, c.blocks),
         "steep": 2.0 ** -rng.integers(0, 100, c.blocks), "zeros": np.where(rng.random(c.blocks) < 0.9, 0, 1),
         "outlier": np.where(np.arange(c.blocks) == 7, 1e30, rng.random(c.blocks)),
         "tiny": rng.integers(0, 1000, c.blocks) * 2.0**-149}[kind]
    v[:] = torch.from_numpy(x.astype(np.float32)).cuda()[:, None, None]
    q = c.make((batch, 2, 64)).abs()
    if kind == "tiny":
        q.fill_(2.0**-140)
    else:
        q.fill_(0.5)
    for keep in (10, 150, 299):
        run_select(c, q, keep, 1, 2)


@pytest.mark.parametrize("batch", [1, 64])
def test_select_ranks_nan_and_infinities(batch):
    blocks = 400
    c = Cache(17, [blocks * 16] * batch, dtype="f32", hkv=1, D=64)
    sort_summaries(c)
    v = c.summary[:, :c.sum_n].view(c.blocks, 2, 64)
    for i, x in ((11, math.nan), (30, math.inf), (50, -math.inf)):
        for b in range(batch):
            v[int(c.tables[b, i]), :, 5] = x
    q = c.make((batch, 1, 64))
    q[:, :, 5] = 1.0
    got = run_select(c, q, 6, 1, 1).cpu().numpy()
    assert (got[:, 0] == 11).any(1).all() and (got[:, 0] == 30).any(1).all()
    q[:, :, 9] = math.nan  # every score is NaN: the lowest blocks
    got = run_select(c, q, 6, 1, 1).cpu().numpy()
    assert (got == [0, 1, 2, 3, 4, 399]).all()


@pytest.mark.parametrize("dtype,D,pad", [("f32", 128, 0), ("f32", 33, 0), ("f32", 200, 0), ("bf16", 80, 0),
                                         ("bf16", 96, 0), ("bf16", 64, 1), ("bf16", 128, 8), ("bf16", 256, 0)])
@pytest.mark.parametrize("blocks,batch", [(300, 3), (1100, 2), (2048 + 3, 1), (2048 + 4, 1), (4100, 1)])
def test_select_where_ctas_share_a_context(dtype, D, pad, blocks, batch):
    """One context next to short ones and an empty one, on either side of what a CTA gathers."""
    ctx = [blocks * 16 - 5] + [64 * 16, 0][:batch - 1]
    c = Cache(20, ctx, dtype=dtype, layers=2, layer=1, hkv=2, D=D, pad=pad)
    sort_summaries(c)
    q = c.make((batch, 8, D))
    for keep, sink, recent in ((40, 1, 2), (3, 1, 2), (64, 0, 0)):  # the second leaves nothing to choose
        run_select(c, q, keep, sink, recent)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("bf16", 80), ("f32", 64), ("f32", 33)])
@pytest.mark.parametrize("blocks", [1500, 5000])
def test_select_short_contexts_in_a_call_for_long_ones(dtype, D, blocks):
    """max_context_len is a bound, as a captured graph has it: most CTAs of a context then have no block."""
    keep = 7
    ctx = [keep * 16 + 1, (keep + 2) * 16, 0, 16 * 16, 1, 300 * 16 + 5]
    c = Cache(24, ctx, dtype=dtype, hkv=2, D=D, pitch=blocks)
    sort_summaries(c)
    q = c.make((len(ctx), 8, D))
    run_select(c, q, keep, 1, 2, max_context_len=blocks * 16)
    run_select(c, q, keep, 0, 0, max_context_len=blocks * 16)
    run_select(c, q, 1, 0, 0, max_context_len=blocks * 16)


@pytest.mark.parametrize("kind", ["equal", "few", "steep", "zeros", "outlier", "tiny", "close", "huge"])
@pytest.mark.parametrize("batch,blocks", [(1, 1500), (1, 2600), (64, 300)])
@pytest.mark.parametrize("D", [64, 128])
def test_select_bf16_where_scores_tie_or_crowd(kind, batch, blocks, D):
    """The 32-bit scores leave more blocks open than one pass can rank, or none that it may trust."""
    torch = _torch()
    c = Cache(21, [blocks * 16] * batch, hkv=1, D=D)
    v = c.summary[:, :c.sum_n].view(c.blocks, 2, D)
    rng = np.random.default_rng(22)
    x = {"equal": np.ones(c.blocks), "few": rng.integers(0, 5, c.blocks),
         "steep": 2.0 ** -rng.integers(0, 100, c.blocks), "zeros": np.where(rng.random(c.blocks) < 0.9, 0, 1),
         "outlier": np.where(np.arange(c.blocks) == 7, 1e30, rng.random(c.blocks)),
         "tiny": rng.integers(0, 100, c.blocks) * 2.0**-133, "close": np.ones(c.blocks),
         "huge": rng.integers(-200, 200, c.blocks) * 2.0**120}[kind]
    v[:] = torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16).cuda()[:, None, None]
    if kind == "close":  # apart by 2^-20 of the sum: far below what its parts could be off by
        v[:, :, 0] = torch.from_numpy(rng.integers(0, 128, c.blocks).astype(np.float32) * 2.0**-20).cuda()[:, None]
    q = c.make((batch, 2, D))
    q.fill_({"tiny": 2.0**-120, "huge": 2.0**100}.get(kind, 0.5))
    for keep in (10, 150, 299):
        run_select(c, q, keep, 1, 2)


@pytest.mark.parametrize("batch,blocks", [(1, 400), (1, 2600), (64, 400)])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_select_bf16_ranks_nan_and_infinities(batch, blocks, D):
    c = Cache(23, [blocks * 16] * batch, hkv=1, D=D)
    sort_summaries(c)
    v = c.summary[:, :c.sum_n].view(c.blocks, 2, D)
    for i, x in ((11, math.nan), (30, math.inf), (50, -math.inf)):
        for b in range(batch):
            v[int(c.tables[b, i]), :, 5] = x
    q = c.make((batch, 1, D))
    q[:, :, 5] = 1.0
    got = run_select(c, q, 6, 1, 1).cpu().numpy()
    assert (got[:, 0] == 11).any(1).all() and (got[:, 0] == 30).any(1).all()
    q[:, :, 7] = math.inf  # finite rows decide by the sign of one channel
    run_select(c, q, 6, 1, 1)
    q[:, :, 9] = math.nan  # every score is NaN: the lowest blocks
    got = run_select(c, q, 6, 1, 1).cpu().numpy()
    assert (got == [0, 1, 2, 3, 4, blocks - 1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset,extra", [(8, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 3), (0, 0, 64)])
def test_select_over_strides_and_alignments(dtype, pad, offset, extra):
    c = Cache(18, [2000, 1, 777], dtype=dtype, hkv=2, D=64, pad=pad, offset=offset)
    sort_summaries(c)
    q = c.make((3, 8 * 64 + extra), offset)[:, :8 * 64].unflatten(1, (8, 64))
    run_select(c, q, 9, 1, 1)


@pytest.mark.parametrize("ctx,bit", [([-1, 800], 4), ([801, 800], 4), ([800, 800], 1)])
def test_select_flags_bad_lengths_and_ids(ctx, bit):
    torch = _torch()
    c = Cache(19, [800, 800], hkv=1, D=64)
    sort_summaries(c)
    want = S.select(np.ones((2, 2, 64)), c.summary64(), c.tables, c.ctx, 16, 0, 1, 5, 1, 1)
    if bit == 1:
        c.tables_d[0, 20:40] = 10**7
    ctx_d = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    q = torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    args, out = c.select_args(q, 5, 1, 1, context_lens=ctx_d.data_ptr())
    assert qvp.select_blocks(args, _stream()) == qvp.OK
    assert c.errors() == bit
    got = out.cpu().numpy()
    assert np.array_equal(got[1], want[1])
    if bit == 4:
        assert (got[0] == -1).all()
    else:
        assert not ((got[0] >= 20) & (got[0] < 40)).any()


# --- attention over the lists ---------------------------------------------------


def near_attention(c, got, q, selected, scale=None, ctx=None, one_term=False):
    q64 = q.double().cpu().numpy()
    scale = np.float64(np.float32(scale or c.D ** -0.5))
    want, size, reach = S.attend(q64, c.pool64(), c.tables, c.ctx if ctx is None else ctx, c.layer, scale, selected)
    tokens = selected.shape[2] * c.T
    weight = (c.D + 4) * 2.0**-23 * reach + 2.0**-21 + tokens * 2.0**-24
    if c.dtype == "bf16":
        weight = weight + (2.0**-8 if one_term else 2.0**-16)
    bound = STEP[c.dtype] * np.abs(want) + 2 * weight[..., None] * size
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


def random_lists(c, keep, sparse=True):
    """Ascending lists of distinct blocks, -1 past their ends."""
    out = np.full((len(c.ctx), c.hkv, keep), -1, dtype=np.int32)
    for b, h in itertools.product(range(len(c.ctx)), range(c.hkv)):
        n = -(-int(c.ctx[b]) // c.T)
        take = min(n, keep)
        out[b, h, :take] = np.sort(c.rng.permutation(n)[:take])
    return out


def run_attend(c, q, lists, **kw):
    torch = _torch()
    selected = torch.from_numpy(lists).cuda()
    args, out = c.attend_args(q, selected, **kw)
    assert qvp.decode_selected(args, _stream()) == qvp.OK, qvp.last_error()
    assert c.errors() == 0
    near_attention(c, out, q, lists, kw.get("scale"), one_term=q.shape[1] // c.hkv > 8)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,D,T", [(28, 4, 128, 16), (8, 2, 64, 16), (5, 1, 96, 8), (6, 3, 80, 32),
                                        (2, 2, 256, 16), (14, 2, 33, 5), (4, 1, 16, 1), (16, 1, 128, 16),
                                        (9, 1, 64, 16), (17, 1, 128, 16), (3, 1, 128, 32), (4, 2, 64, 48),
                                        (1, 1, 128, 16), (20, 2, 256, 16)])
@pytest.mark.parametrize("keep", [1, 7, 40])
def test_attend_matches_the_definition(dtype, hq, hkv, D, T, keep):
    ctx = [1, 0, T, T + 1, 13 * T - 1, 90 * T, 41 * T + 1]
    c = Cache(20, ctx, dtype=dtype, layers=2, layer=1, T=T, hkv=hkv, D=D)
    run_attend(c, c.make((len(ctx), hq, D)), random_lists(c, keep))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,keep", [(1, 128), (1, 1000), (3, 130), (40, 64), (300, 9)])
def test_attend_over_batches_and_long_lists(dtype, batch, keep):
    rng = np.random.default_rng(21)
    ctx = rng.integers(1, 1200 * 16 if batch < 10 else 2000, size=batch)
    ctx[0] = 1100 * 16 - 5
    c = Cache(22, ctx, dtype=dtype, hkv=2, D=64)
    run_attend(c, c.make((batch, 14, 64)), random_lists(c, keep))


def test_attend_takes_lists_in_any_order_with_gaps_and_repeats():
    torch = _torch()
    c = Cache(23, [500, 333, 16], hkv=2, D=128)
    lists = np.full((3, 2, 12), -1, dtype=np.int32)
    lists[0, 0, [1, 4, 11]] = [31, 0, 7]
    lists[0, 1, 3:6] = [5, 5, 9]          # block 5 counts twice
    lists[1, 0, ::2] = [20, 1, 19, 2, 18, 3]
    lists[2, 0, 11] = 0                    # the other list of this sequence is empty
    run_attend(c, c.make((3, 8, 128)), lists)
    lists[:] = -1
    lists[:, :, 3] = -5
    out = run_attend(c, c.make((3, 8, 128)), lists)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset,extra", [(8, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 3), (0, 0, 64), (64, 2, 2)])
def test_attend_over_strides_and_alignments(dtype, pad, offset, extra):
    c = Cache(24, [300, 77, 16, 1], dtype=dtype, hkv=2, D=64, pad=pad, offset=offset)
    q = c.make((4, 8 * 64 + extra), offset)[:, :8 * 64].unflatten(1, (8, 64))
    run_attend(c, q, random_lists(c, 6))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_attend_large_scores_and_stale_slots(dtype, D):
    """Maxima that jump from block to block, and NaN in every slot past the contexts."""
    torch = _torch()
    c = Cache(25, [300, 77, 16, 1, 170], dtype=dtype, hkv=2, D=D)
    view = c.pool[:, :c.n].view(c.blocks, 2, 16, 2, D)
    used = torch.zeros(c.blocks, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.ctx):
        for j in range(-(-int(n) // 16)):
            used[int(c.tables[b, j]), :min(16, int(n) - j * 16)] = True
    view.masked_fill_(~used[:, None, :, None, None], math.nan)
    q = c.make((5, 8, D), scale=24.0)
    torch.nan_to_num_(c.pool[:, c.n:])
    lists = random_lists(c, 20)
    selected = torch.from_numpy(lists).cuda()
    args, out = c.attend_args(q, selected)
    assert qvp.decode_selected(args, _stream()) == qvp.OK and c.errors() == 0
    assert torch.isfinite(out).all()
    near_attention(c, out, q, lists)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("bf16", 64), ("f32", 64), ("bf16", 96)])
def test_attend_scores_of_minus_infinity(dtype, D):
    """Blocks whose scores are all -inf weigh nothing; alone they give NaN, as a softmax over them does."""
    torch = _torch()
    c = Cache(26, [160, 160], dtype=dtype, hkv=1, D=D)
    view = c.pool[:, :c.n].view(c.blocks, 2, 16, 1, D)
    q = c.make((2, 4, D)).abs() + 0.1
    for j in range(9):
        view[int(c.tables[0, j]), 0, :, :, 3] = -math.inf
    view[c.tables_d[1].long(), 0, :, :, 3] = -math.inf
    lists = np.broadcast_to(np.arange(10, dtype=np.int32), (2, 1, 10)).copy()
    args, out = c.attend_args(q, torch.from_numpy(lists).cuda())
    assert qvp.decode_selected(args, _stream()) == qvp.OK and c.errors() == 0
    assert torch.isnan(out[1]).all()
    lists[0, 0, :9] = -1
    near_attention(c, out[:1], q[:1], lists[:1], ctx=c.ctx[:1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,hq", [(64, 4), (96, 4), (128, 8), (128, 16), (80, 4), (33, 2)])
def test_attend_infinities_and_nan_stay_where_they_are(dtype, D, hq):
    """An infinity or NaN of V reaches its dimension of the heads that attend it, and no other."""
    torch = _torch()
    c = Cache(36, [160, 320, 160], dtype=dtype, hkv=1, D=D)
    q = c.make((3, hq, D))
    clean = np.broadcast_to(np.arange(10, dtype=np.int32), (3, 1, 10)).copy()
    args, out = c.attend_args(q, torch.from_numpy(clean).cuda())
    assert qvp.decode_selected(args, _stream()) == qvp.OK
    want = out.double().cpu().numpy()
    v = c.pool[:, :c.n].unflatten(1, (2, 16, 1, D))[:, 1]
    for block, slot, dim, x in ((0, 3, 1, math.inf), (4, 15, 5, -math.inf), (7, 0, D - 1, math.nan)):
        v[int(c.tables[0, block]), slot, 0, dim] = x
        want[0, :, dim] = x
    v[int(c.tables[1, 15]), :, 0, 2] = math.inf  # not listed
    assert qvp.decode_selected(args, _stream()) == qvp.OK and c.errors() == 0
    got = out.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    # both results of a finite element are within the bound of the same exact value: weights of one bf16 term,
    # values below 6, and the rounding of each result
    assert np.abs(got[fine] - want[fine]).max() < (2 * (2.0**-8 + 2.0**-9) * 6 if dtype == "bf16" else 1e-4)


@pytest.mark.parametrize("what,bit", [("past", 1), ("id", 1), ("long", 4), ("negative", 4)])
@pytest.mark.parametrize("D", [128, 96])
def test_attend_flags_bad_entries_and_serves_the_rest(what, bit, D):
    torch = _torch()
    c = Cache(27, [160, 160], hkv=2, D=D)
    q = c.make((2, 4, D))
    lists = random_lists(c, 6)
    want, _, _ = S.attend(q.double().cpu().numpy(), c.pool64(), c.tables, c.ctx, 0, D ** -0.5, lists)
    selected = torch.from_numpy(lists).cuda()
    ctx = [160, 160]
    if what == "past":
        selected[0, :, 2], selected[0, :, 3] = 10, 2**31 - 1
    elif what == "id":
        c.tables_d[0, :] = torch.tensor([-1, 2**31 - 1] * 5, dtype=torch.int32)
    else:
        ctx[0] = 161 if what == "long" else -3
    ctx_d = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    args, out = c.attend_args(q, selected, context_lens=ctx_d.data_ptr())
    assert qvp.decode_selected(args, _stream()) == qvp.OK
    assert c.errors() == bit
    got = out.double().cpu().numpy()
    assert np.abs(got[1] - want[1]).max() < 2e-2
    if bit == 4:
        assert (got[0] == -7).all()
    elif what == "id":
        assert (got[0] == 0).all()  # every frame is outside the pool: no token is left
    else:
        lists[0, :, 2:4] = -1
        want, _, _ = S.attend(q.double().cpu().numpy(), c.pool64(), c.tables, c.ctx, 0, D ** -0.5, lists)
        assert np.abs(got[0] - want[0]).max() < 2e-2


def test_attend_gives_the_same_bits_from_call_to_call():
    torch = _torch()
    for dtype, hq in (("bf16", 14), ("f32", 14), ("bf16", 32)):
        c = Cache(28, [9000, 40, 3000], dtype=dtype, hkv=2, D=128)
        q = c.make((3, hq, 128))
        selected = torch.from_numpy(random_lists(c, 100)).cuda()
        args, out = c.attend_args(q, selected)
        first = None
        for _ in range(5):
            out.fill_(0)
            assert qvp.decode_selected(args, _stream()) == qvp.OK
            got = _bits(out)
            assert first is None or np.array_equal(got, first)
            first = got


# --- the calls together -----------------------------------------------------------


def chain(c, hq, keep, sink, recent, new, k, v, q_in, freq, pos, sections, lists, q_out, out, stream):
    common = c.common()
    calls = [
        (qvp.rope_append, qvp.rope_append_args(
            **common, **c.at_pool(), **c.at_summary(), num_query_heads=hq, max_query_len=q_in.shape[1],
            query_lens=new.data_ptr(), query=q_in.data_ptr(), key=k.data_ptr(), value=v.data_ptr(),
            query_out=q_out.data_ptr(), rotary_dim=c.D, inv_freq=freq.data_ptr(), rope_positions=pos.data_ptr(),
            rope_sections=sections)),
        (qvp.select_blocks, qvp.select_args(
            **common, **c.at_summary(), num_query_heads=hq, max_context_len=c.pitch * c.T, query=q_out.data_ptr(),
            max_selected=keep, sink_blocks=sink, recent_blocks=recent, selected=lists.data_ptr())),
        (qvp.decode_selected, qvp.decode_selected_args(
            **common, **c.at_pool(), num_query_heads=hq, scale=c.D ** -0.5, query=q_out.data_ptr(),
            selected=lists.data_ptr(), max_selected=keep, out=out.data_ptr()))]

    def step():
        for fn, args in calls:
            assert fn(args, stream()) == qvp.OK, qvp.last_error()
    return step


@pytest.mark.parametrize("how", ["default stream", "another stream", "graph"])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64)])
def test_prompt_then_decode_steps(how, dtype, D):
    """Prompts, then single tokens: each step's lists and outputs follow from the cache that the calls made."""
    torch = _torch()
    B, hq, hkv, keep, sink, recent = 3, 8, 2, 6, 1, 2
    c = Cache(29, [400, 150, 31], dtype=dtype, hkv=hkv, D=D, pitch=30, fill=0.0)
    # room for the steps: every row of the table is mapped
    c.blocks = B * 30 + 2
    ids = c.rng.permutation(c.blocks)[:B * 30].reshape(B, 30).astype(np.int32)
    c.tables[:] = ids
    c.tables_d.copy_(torch.from_numpy(ids))
    c.pool, c.summary = c.make((c.blocks, c.stride), scale=0.0), c.make((c.blocks, c.sum_stride), scale=0.0)
    sections = [D // 8, D // 8, D // 4]
    freq = torch.from_numpy((1e6 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)).cuda()
    stream = torch.cuda.Stream() if how == "another stream" else torch.cuda.current_stream()
    torch.cuda.synchronize()

    # the prompts, in two chunks
    most = 300
    for ctx, new in (([300, 100, 1], [300, 100, 1]), ([400, 150, 31], [100, 50, 30])):
        c.ctx[:] = ctx
        c.ctx_d.copy_(torch.from_numpy(c.ctx))
        new_d = torch.tensor(new, dtype=torch.int32, device="cuda")
        q, k, v = c.make((B, most, hq, D)), c.make((B, most, hkv, D)), c.make((B, most, hkv, D))
        q_out = torch.zeros_like(q)
        pos = torch.arange(most, device="cuda", dtype=torch.int32).expand(3, B, most) + (c.ctx_d - new_d)[None, :, None]
        pos = pos.contiguous()
        args = qvp.rope_append_args(
            **c.common(), **c.at_pool(), **c.at_summary(), num_query_heads=hq, max_query_len=most,
            query_lens=new_d.data_ptr(), query=q.data_ptr(), key=k.data_ptr(), value=v.data_ptr(),
            query_out=q_out.data_ptr(), rotary_dim=D, inv_freq=freq.data_ptr(), rope_positions=pos.data_ptr(),
            rope_sections=sections)
        torch.cuda.synchronize()
        assert qvp.rope_append(args, stream.cuda_stream) == qvp.OK
    torch.cuda.synchronize()
    # what the append wrote is what summarize makes of the pool
    made = c.summary.clone()
    c.summarize()
    torch.cuda.synchronize()
    assert torch.equal(made, c.summary)

    q, k, v = (torch.empty((B, 1, h, D), dtype=_dtype(dtype), device="cuda") for h in (hq, hkv, hkv))
    new_d = torch.ones(B, dtype=torch.int32, device="cuda")
    pos = torch.zeros(3, B, 1, dtype=torch.int32, device="cuda")
    lists = torch.zeros(B, hkv, keep, dtype=torch.int32, device="cuda")
    q_out, out = torch.zeros_like(q), torch.zeros(B, hq, D, dtype=_dtype(dtype), device="cuda")
    step = chain(c, hq, keep, sink, recent, new_d, k, v, q, freq, pos, sections, lists, q_out, out,
                 lambda: torch.cuda.current_stream().cuda_stream)
    graph = None
    for i in range(5):
        c.ctx += 1
        c.ctx_d.copy_(torch.from_numpy(c.ctx))
        for x in (q, k, v):
            x.copy_(c.make(tuple(x.shape)))
        pos[:] = c.ctx_d[None, :, None] - 1
        torch.cuda.synchronize()
        if how == "graph":
            if graph is None:
                step()  # loads the kernels outside the capture
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        else:
            with torch.cuda.stream(stream):
                step()
        assert c.errors() == 0
        q64 = q_out[:, 0].double().cpu().numpy()
        want = S.select(q64, c.summary64(), c.tables, c.ctx, 16, 0, hkv, keep, sink, recent)
        assert np.array_equal(lists.cpu().numpy(), want)
        near_attention(c, out, q_out[:, 0], want)
    if graph is not None:
        del graph


def test_lists_of_every_block_give_the_dense_decode():
    """With room for all blocks the three calls are qvp_decode."""
    torch = _torch()
    c = Cache(30, [500, 37, 300, 1], hkv=4, D=128)
    q = c.make((4, 28, 128))
    args, lists = c.select_args(q, 40, 1, 1)
    assert qvp.select_blocks(args, _stream()) == qvp.OK
    args, out = c.attend_args(q, lists)
    assert qvp.decode_selected(args, _stream()) == qvp.OK
    dense = torch.zeros_like(out)
    a = qvp.decode_args(**{k: v for k, v in c.common().items()}, pool=c.pool.data_ptr(), block_stride=c.stride * 2,
                        num_query_heads=28, scale=128 ** -0.5, max_context_len=500, query=q.data_ptr(),
                        out=dense.data_ptr())
    plan = qvp.decode_plan(a)
    ws = torch.empty(plan["workspace_bytes"], dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert qvp.decode(a, _stream()) == qvp.OK
    assert c.errors() == 0
    assert (out.float() - dense.float()).abs().max() < 2e-2
    near_attention(c, out, q, lists.cpu().numpy())


def test_two_graphs_and_two_streams_share_nothing():
    """Calls that run at the same time keep their own results: there is no hidden workspace."""
    torch = _torch()
    caches = [Cache(31 + i, [3000 + 500 * i, 200, 1700], hkv=2, D=128) for i in range(2)]
    work = []
    for c in caches:
        sort_summaries(c)
        q = c.make((3, 14, 128))
        sargs, lists = c.select_args(q, 20, 1, 1)
        aargs, out = c.attend_args(q, lists)
        work.append((c, q, sargs, lists, aargs, out))
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in work]
    for c, q, sargs, lists, aargs, out in work:
        assert qvp.select_blocks(sargs, _stream()) == qvp.OK and qvp.decode_selected(aargs, _stream()) == qvp.OK
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            assert qvp.select_blocks(sargs, _stream()) == qvp.OK
            assert qvp.decode_selected(aargs, _stream()) == qvp.OK
        graphs.append(g)
        lists.fill_(-1), out.fill_(0)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, q, sargs, lists, aargs, out in work:
        want = S.select(q.double().cpu().numpy(), c.summary64(), c.tables, c.ctx, 16, 0, 2, 20, 1, 1)
        assert c.errors() == 0 and np.array_equal(lists.cpu().numpy(), want)
        near_attention(c, out, q, want)


def test_summaries_move_with_the_block_movers():
    """A copy of a block and of its summary, by the same pairs, is a summarized copy."""
    torch = _torch()
    c = Cache(33, [160], hkv=2, D=64, spare=12)
    c.summarize()
    free = np.setdiff1d(np.arange(c.blocks), c.tables[0])[:10].astype(np.int32)
    pairs = torch.from_numpy(np.stack((c.tables[0], free), 1).reshape(-1)).cuda()
    summary_bytes = qvp.block_bytes(qvp.summary_shape(c.shape))
    for base, stride, nbytes in ((c.pool, c.stride * 2, qvp.block_bytes(c.shape)),
                                 (c.summary, c.sum_stride * 2, summary_bytes)):
        assert qvp.lib.qvp_copy_blocks(base.data_ptr(), stride, c.blocks, nbytes, pairs.data_ptr(), 10,
                                       c.error.data_ptr(), _stream()) == qvp.OK
    moved = c.summary.clone()
    c.tables[0], c.tables_d[0] = free, torch.from_numpy(free).cuda()
    c.summarize()
    assert c.errors() == 0 and torch.equal(moved, c.summary)


@pytest.mark.parametrize("op", ["append", "summarize", "select", "attend"])
def test_the_measured_cases_flag_nothing(op):
    """The calls of perf/operators.py, its listed cases and drawn ones, leave their error words at zero."""
    torch = _torch()
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("measured_operators", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    rng = random.Random(42)
    cases = m.listed() + [m.draw(rng) for _ in range(24)]
    for i, case in enumerate(c for c in cases if c["op"] == op):
        state = m.prepare(case, i)
        m.run(state)
        torch.cuda.synchronize()
        assert int(state["error"].item()) == 0, case
        del state
    torch.cuda.empty_cache()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the last blocks are read and written where they are."""
    torch = _torch()
    shape = qvp.make_shape(16, 1, 8, 128, 2)
    stride = qvp.block_stride(shape) // 2
    blocks = (1 << 32) // stride + 64
    free, _ = torch.cuda.mem_get_info()
    if free < blocks * stride * 2 + (4 << 30):
        pytest.skip("not enough device memory")
    c = Cache(34, [64 * 16], hkv=8, D=128)
    c.blocks = blocks
    c.tables = np.arange(blocks - 64, blocks, dtype=np.int32)[None, :].copy()
    c.tables_d.copy_(torch.from_numpy(c.tables))
    c.pool = torch.zeros(blocks, stride, dtype=torch.bfloat16, device="cuda")
    c.summary = torch.zeros(blocks, c.sum_stride, dtype=torch.bfloat16, device="cuda")
    k, v = c.make((1, 1024, 8, 128)), c.make((1, 1024, 8, 128))
    new = torch.tensor([1024], dtype=torch.int32, device="cuda")
    args = qvp.rope_append_args(**c.common(), **c.at_pool(), **c.at_summary(), num_query_heads=0, max_query_len=1024,
                                query_lens=new.data_ptr(), key=k.data_ptr(), value=v.data_ptr())
    assert qvp.rope_append(args, _stream()) == qvp.OK
    torch.cuda.synchronize()
    tail = c.pool[blocks - 64:].view(64, 2, 16, 8, 128)
    assert torch.equal(tail[:, 0].reshape(1024, 8, 128), k[0]) and torch.equal(tail[:, 1].reshape(1024, 8, 128), v[0])
    assert int(c.pool[:blocks - 64].count_nonzero()) == 0
    q = c.make((1, 64, 128))
    sargs, lists = c.select_args(q, 9, 1, 1)
    aargs, out = c.attend_args(q, lists)
    assert qvp.select_blocks(sargs, _stream()) == qvp.OK and qvp.decode_selected(aargs, _stream()) == qvp.OK
    assert c.errors() == 0
    # the same cache in a small pool
    d = Cache(35, [64 * 16], hkv=8, D=128, spare=0)
    d.tables = np.arange(64, dtype=np.int32)[None, :].copy()
    d.tables_d.copy_(torch.from_numpy(d.tables))
    d.pool, d.summary = c.pool[blocks - 64:].clone(), c.summary[blocks - 64:].clone()
    want = S.select(q.double().cpu().numpy(), d.summary64(), d.tables, d.ctx, 16, 0, 8, 9, 1, 1)
    assert np.array_equal(lists.cpu().numpy(), want)
    near_attention(d, out, q, want)
    del c, tail
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,D,T", [("bf16", 64, 48), ("bf16", 128, 256), ("f32", 64, 48), ("f32", 80, 256)])
def test_the_longest_context(dtype, D, T):
    """2^31 - 1 tokens: the last block's slots end past 31 bits."""
    torch = _torch()
    longest = 2**31 - 1
    last = (longest - 1) // T
    c = Cache(36, [6 * T], dtype=dtype, hkv=1, D=D, T=T, spare=0)
    k, v = c.make((1, 5, 1, D)), c.make((1, 5, 1, D))
    c.pitch, c.ctx = last + 1, np.array([longest], dtype=np.int32)
    c.ctx_d.fill_(longest)
    c.tables_d = torch.full((1, c.pitch), -1, dtype=torch.int32, device="cuda")
    c.tables_d[0, 0], c.tables_d[0, last - 1], c.tables_d[0, last] = 5, 1, 2
    new = torch.tensor([5], dtype=torch.int32, device="cuda")
    freq = torch.tensor([2.0**-k for k in range(16)], device="cuda")  # exact angles
    before = c.pool64()
    args = qvp.rope_append_args(**c.common(), **c.at_pool(), **c.at_summary(), num_query_heads=0, max_query_len=5,
                                query_lens=new.data_ptr(), key=k.data_ptr(), value=v.data_ptr(), rotary_dim=32,
                                inv_freq=freq.data_ptr())
    assert qvp.rope_append(args, _stream()) == qvp.OK, qvp.last_error()
    assert c.errors() == 0
    after, k64, v64 = c.pool64(), k.double().cpu().numpy()[0, :, 0], v.double().cpu().numpy()[0, :, 0]
    want = before.copy()
    filled = longest - last * T
    for t in range(5):
        at = longest - 5 + t
        x, y = k64[t, :16].copy(), k64[t, 16:32].copy()
        angle = np.array([math.fmod(at * 2.0**-j, 2 * math.pi) for j in range(16)])
        row = k64[t].copy()
        row[:16], row[16:32] = x * np.cos(angle) - y * np.sin(angle), y * np.cos(angle) + x * np.sin(angle)
        block, slot = (2, at - last * T) if at >= last * T else (1, at - (last - 1) * T)
        want[block, 0, 0, slot, 0], want[block, 0, 1, slot, 0] = row, v64[t]
    # the angle in turns is a 64-bit product below 2^29: off by 2^-25 of a turn, 2^-22 of an element's pair
    size = np.zeros_like(want)
    size[..., :16] = size[..., 16:32] = np.abs(want[..., :16]) + np.abs(want[..., 16:32])
    assert (np.abs(after - want) <= STEP[dtype] * np.abs(want) + 2.0**-19 * size).all()
    assert np.array_equal(c.summary64()[2, 0], S.summary_of(after, 2, 0, filled))
    lists = np.array([[[0, last - 1, last]]], dtype=np.int32)
    q = c.make((1, 4, D))
    args, out = c.attend_args(q, torch.from_numpy(lists).cuda())
    assert qvp.decode_selected(args, _stream()) == qvp.OK, qvp.last_error()
    assert c.errors() == 0
    # the same blocks as a short context
    c.ctx, c.tables = np.array([2 * T + filled]), np.array([[5, 1, 2]])
    near_attention(c, out, q, np.array([[[0, 1, 2]]], dtype=np.int32))
