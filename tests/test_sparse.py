"""CPU checks of the sparse-attention calls: what they refuse before any launch,
the summary pool's shape, and the 64-bit oracle against the dense one."""
import ctypes as C

import numpy as np
import pytest

import oracle
import qvp
import sparse_oracle as S
import workloads as W

SHAPE = qvp.make_shape(16, 2, 2, 64, 2)
STRIDE = qvp.block_stride(SHAPE)
SUM_STRIDE = qvp.block_stride(qvp.summary_shape(SHAPE))


def _cache(**kw):
    base = dict(shape=SHAPE, dtype=qvp.DTYPE_BF16, layer=1, num_blocks=8, batch=2, max_blocks_per_seq=4,
                block_tables=0x2000, context_lens=0x3000)
    base.update(kw)
    return base


def _append(**kw):
    base = dict(_cache(), pool=0x1000, block_stride=STRIDE, num_query_heads=4, max_query_len=5, query_lens=0x4000,
                query=0x5000, key=0x6000, value=0x7000, query_out=0x8000, rotary_dim=64, inv_freq=0x9000,
                rope_positions=0xa000, rope_sections=[8, 12, 12], summary=0xb000, summary_stride=SUM_STRIDE)
    base.update(kw)
    return qvp.rope_append(qvp.rope_append_args(**base))


def _summarize(**kw):
    base = dict(_cache(), pool=0x1000, block_stride=STRIDE, max_context_len=64, summary=0xb000,
                summary_stride=SUM_STRIDE)
    base.update(kw)
    return qvp.summarize_blocks(qvp.summarize_args(**base))


def _select(**kw):
    base = dict(_cache(), summary=0xb000, summary_stride=SUM_STRIDE, num_query_heads=4, max_context_len=64,
                query=0x5000, max_selected=3, sink_blocks=1, recent_blocks=1, selected=0xc000)
    base.update(kw)
    return qvp.select_blocks(qvp.select_args(**base))


def _attend(**kw):
    base = dict(_cache(), pool=0x1000, block_stride=STRIDE, num_query_heads=4, scale=0.125, query=0x5000,
                selected=0xc000, max_selected=3, out=0xd000)
    base.update(kw)
    return qvp.decode_selected(qvp.decode_selected_args(**base))


COMMON = [
    dict(shape=qvp.make_shape(0, 2, 2, 64, 2)),
    dict(shape=qvp.make_shape(16, 2, 2, 64, 4)),          # element size of the other type
    dict(dtype=7),
    dict(layer=2),
    dict(num_blocks=0),
    dict(max_blocks_per_seq=0),
    dict(block_tables=0),
    dict(context_lens=0),
]
POOL = [dict(pool=0), dict(block_stride=STRIDE - 2), dict(pool=0x1001)]
SUMMARY = [dict(summary_stride=SUM_STRIDE - 2), dict(summary=0xb001)]


@pytest.mark.parametrize("bad", COMMON + POOL + SUMMARY + [
    dict(num_query_heads=3),
    dict(rotary_dim=63),
    dict(rotary_dim=66),
    dict(rope_sections=[8, 12, 11]),                      # 31 pairs of 32
    dict(rope_sections=[]),                               # positions without axes
    dict(rope_sections=[2**31, 2**31, 32]),               # a sum that wraps to 32 in 32 bits
    dict(inv_freq=0),
    dict(query_lens=0),
    dict(query=0),
    dict(query_out=0),
    dict(key=0),
    dict(value=0),
    dict(max_query_len=0),
    dict(query_pitch=4 * 64 - 1),
    dict(key_pitch=2 * 64 - 1),
    dict(value_pitch=2 * 64 - 1),
    dict(query_out=0x5000, query_pitch=8 * 64),           # in place over rows that are not dense
    dict(key=0x6001),
])
def test_rope_append_refuses_inconsistent_arguments(bad):
    assert _append(**bad) == qvp.ERR_INVALID
    assert qvp.last_error()


@pytest.mark.parametrize("bad", COMMON + POOL + SUMMARY + [
    dict(summary=0), dict(max_context_len=0), dict(max_context_len=65)])
def test_summarize_refuses_inconsistent_arguments(bad):
    assert _summarize(**bad) == qvp.ERR_INVALID
    assert qvp.last_error()


@pytest.mark.parametrize("bad", COMMON + SUMMARY + [
    dict(summary=0), dict(max_context_len=0), dict(max_context_len=65), dict(num_query_heads=0),
    dict(num_query_heads=5), dict(max_selected=0), dict(sink_blocks=2, recent_blocks=2),
    dict(sink_blocks=2**32 - 1, recent_blocks=2), dict(query=0), dict(selected=0), dict(query_pitch=255),
    dict(query=0x5001)])
def test_select_refuses_inconsistent_arguments(bad):
    assert _select(**bad) == qvp.ERR_INVALID
    assert qvp.last_error()


@pytest.mark.parametrize("bad", COMMON + POOL + [
    dict(num_query_heads=0), dict(num_query_heads=5), dict(max_selected=0), dict(query=0), dict(selected=0),
    dict(out=0), dict(out=0xd001), dict(query_pitch=255)])
def test_decode_selected_refuses_inconsistent_arguments(bad):
    assert _attend(**bad) == qvp.ERR_INVALID
    assert qvp.last_error()


@pytest.mark.parametrize("call,arrays", [(_append, ["query_lens", "inv_freq", "rope_positions"]),
                                         (_summarize, ["first_tokens"]), (_select, ["selected"]),
                                         (_attend, ["selected"])])
def test_misaligned_arrays_are_refused(call, arrays):
    for name in arrays + ["block_tables", "context_lens", "error_word"]:
        for off in (1, 2):
            assert call(**{name: 0xe000 + off}) == qvp.ERR_INVALID, name
            assert "aligned" in qvp.last_error()


@pytest.mark.parametrize("call", [_append, _summarize, _select, _attend])
def test_what_the_kernels_do_not_cover_is_refused(call):
    wide = qvp.make_shape(16, 2, 2, 264, 2)
    assert call(shape=wide) == qvp.ERR_UNSUPPORTED
    assert call(batch=65536) == qvp.ERR_UNSUPPORTED
    assert call(batch=0) == qvp.OK  # nothing to do: no launch


@pytest.mark.parametrize("call,pool", [(_append, True), (_summarize, True), (_select, False), (_attend, True)])
def test_blocks_past_32_bits_of_elements_are_refused(call, pool):
    huge = qvp.make_shape(65536, 1, 512, 128, 2)
    where = dict(block_stride=qvp.block_stride(huge)) if pool else {}
    if call is not _attend:
        where["summary_stride"] = qvp.block_stride(qvp.summary_shape(huge))
    if call is not _summarize:
        where["num_query_heads"] = 512
    assert call(shape=huge, layer=0, **where) == qvp.ERR_UNSUPPORTED
    assert "elements" in qvp.last_error()


@pytest.mark.parametrize("call", [_append, _summarize, _select])
def test_summaries_past_32_bits_of_rows_are_refused(call):
    # 2^31 layers of 2 kv heads; the layers alone still fit the shape
    deep = qvp.make_shape(1, 2**31, 2, 8, 2)
    where = {} if call is _select else dict(block_stride=qvp.block_stride(deep))
    if call is _append:
        where.update(rotary_dim=8, rope_sections=[1, 1, 2])
    for stride in (8, 256, 2**37, 2**63):  # none is a summary block's size
        assert call(shape=deep, layer=0, num_blocks=1, summary_stride=stride, **where) == qvp.ERR_UNSUPPORTED
        assert "layer" in qvp.last_error()


@pytest.mark.parametrize("call", [_append, _attend])
def test_blocks_whose_size_wraps_are_refused(call):
    # 2^16 tokens x 2^31 layers x 2^6 heads x 2^8 elements x K and V x 4 bytes = 2^64: any stride would do
    wraps = qvp.make_shape(65536, 2**31, 64, 256, 4)
    assert qvp.block_bytes(wraps) == 0
    where = dict(summary=0, rotary_dim=0, max_query_len=1) if call is _append else {}
    assert call(shape=wraps, layer=2**30, dtype=qvp.DTYPE_F32, num_query_heads=64, block_stride=256,
                **where) == qvp.ERR_UNSUPPORTED


@pytest.mark.parametrize("call,stride", [(_append, "block_stride"), (_append, "summary_stride"),
                                         (_summarize, "block_stride"), (_summarize, "summary_stride"),
                                         (_select, "summary_stride"), (_attend, "block_stride")])
def test_pools_whose_size_wraps_are_refused(call, stride):
    assert call(num_blocks=2**30, **{stride: 2**34}) == qvp.ERR_UNSUPPORTED
    assert "bytes" in qvp.last_error()


def test_select_refuses_contexts_that_do_not_fit_a_cluster():
    blocks = 8 * 20480 + 2
    assert _select(max_blocks_per_seq=blocks + 1, max_context_len=(blocks + 1) * 16) == qvp.ERR_UNSUPPORTED


@pytest.mark.parametrize("sink,recent", [(1, 1), (0, 0), (0, 3)])
def test_select_refuses_one_block_past_its_longest_context(sink, recent):
    # 114,688 blocks between sink and recent are served; the GPU tests launch that many
    blocks = 114688 + sink + recent + 1
    for tokens in (16, 1):
        shape = qvp.make_shape(tokens, 2, 2, 64, 2)
        assert _select(shape=shape, sink_blocks=sink, recent_blocks=recent, max_blocks_per_seq=blocks,
                       max_context_len=(blocks - 1) * tokens + 1) == qvp.ERR_UNSUPPORTED
        assert "114688" in qvp.last_error()


@pytest.mark.parametrize("call", [_select, _attend])
@pytest.mark.parametrize("entries", [2**31, 2**32 - 1])
def test_lists_past_31_bits_are_refused(call, entries):
    assert call(max_selected=entries) == qvp.ERR_UNSUPPORTED


@pytest.mark.parametrize("fn", ["qvp_rope_append", "qvp_summarize_blocks", "qvp_select_blocks", "qvp_decode_selected"])
def test_null_arguments_are_refused(fn):
    assert getattr(qvp.lib, fn)(None, None) == qvp.ERR_INVALID


def test_summary_shape_is_one_row_pair_per_layer_and_head():
    s = qvp.summary_shape(qvp.make_shape(16, 3, 4, 128, 2))
    assert (s.tokens_per_block, s.num_layers, s.num_kv_heads, s.head_dim, s.bytes_per_element) == (1, 12, 1, 128, 2)
    assert qvp.block_bytes(s) == 3 * 4 * 2 * 128 * 2
    assert qvp.lib.qvp_summary_shape(None, C.byref(s)) == qvp.ERR_INVALID
    assert qvp.lib.qvp_summary_shape(C.byref(s), None) == qvp.ERR_INVALID


def test_too_many_rotary_axes_are_refused():
    with pytest.raises(ValueError):
        _append(rope_sections=[8, 8, 8, 4, 4])


def _random_cache(seed, layers=2, T=8, hkv=2, D=16, blocks=40):
    rng = np.random.default_rng(seed)
    pool = rng.standard_normal((blocks, layers, 2, T, hkv, D)).astype(np.float32).astype(np.float64)
    summary = np.stack((pool[:, :, 0].min(2), pool[:, :, 0].max(2)), axis=3)
    return rng, pool, summary


def test_the_oracle_over_every_block_is_the_dense_oracle():
    w = W.small(5, batch=3, ctx_lo=20, ctx_hi=150, hq=6, hkv=2, head_dim=32, dtype="f32")
    raw, q = W.host_inputs(w)
    dense, _ = oracle.port_decode(w, raw, q)
    pool = raw.reshape(w.num_blocks, -1)[:, :w.block_bytes].copy().view(np.float32).astype(np.float64)
    pool = pool.reshape(w.num_blocks, 1, 2, 16, 2, 32)
    lists = np.broadcast_to(np.arange(w.pitch), (3, 2, w.pitch))
    out, _, _ = S.attend(q, pool, w.tables, w.context_lens, 0, w.scale, lists)
    assert np.max(np.abs(out - dense)) < 1e-5 * np.max(np.abs(dense))


def test_no_token_exceeds_its_blocks_score():
    rng, pool, summary = _random_cache(1)
    tables = rng.permutation(40)[:20].reshape(2, 10)
    q = rng.standard_normal((2, 6, 16))
    for b in range(2):
        for h in range(2):
            s = S.scores(q, summary, tables, b, 10, 1, h, 3)
            products = pool[tables[b], 1, 0, :, h] @ q[b, 3 * h:3 * h + 3].sum(0)
            assert (products.max(1) <= s + 1e-12).all()


def test_the_oracle_keeps_sink_recent_and_the_lowest_of_equal_blocks():
    _, pool, summary = _random_cache(2)
    summary[:] = summary[:1]  # every block scores the same
    q = np.random.default_rng(0).standard_normal((1, 2, 16))
    got = S.select(q, summary, np.arange(40)[None, :], [317], 8, 0, 2, 7, 1, 2)
    assert got.tolist() == [[[0, 1, 2, 3, 4, 38, 39]] * 2]


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_oracle_rotation_depends_on_the_distance_alone(interleaved):
    rng = np.random.default_rng(3)
    q, k, f = rng.standard_normal(16), rng.standard_normal(16), 10.0 ** -np.arange(6)
    a = S.rotate(q, [9], f, [6], interleaved) @ S.rotate(k, [4], f, [6], interleaved)
    b = S.rotate(q, [105], f, [6], interleaved) @ S.rotate(k, [100], f, [6], interleaved)
    assert abs(a - b) < 1e-12
    assert (S.rotate(q, [9], f, [6], interleaved)[12:] == q[12:]).all()
