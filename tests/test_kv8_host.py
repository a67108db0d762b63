"""Refusals of the 8-bit cache entry points (host checks, no GPU needed) and the plain
quantiser that the GPU tests compare with."""
import numpy as np
import pytest

import fa_dec
import kv8_plain as P

INVALID = fa_dec.FA_ERR_INVALID_ARG
CAPACITY = fa_dec.FA_ERR_CAPACITY
A = 0x1000   # an aligned address that is never dereferenced: every call here is refused on the host


def append(**o):
    a = dict(k=A, v=A, src_type=1, row_stride=1024, M=1, n_layers=1, n_kv_heads=8, pos=A, slot=A, bt=A, bt_stride=4,
             n_pages=4, fmt=0, pool=A)
    a.update(o)
    fa_dec.op_kv8_append(**a)


def qkv_append(**o):
    a = dict(qkv=A, M=1, n_heads=16, n_kv_heads=8, pos=A, slot=A, bt=A, bt_stride=4, n_pages=4, qn=A, kn=A, eps=1e-5,
             rope=A, max_pos=64, fmt=0, pool=A, q_out=A)
    a.update(o)
    fa_dec.op_qknorm_rope_append_kv8(**a)


def gather(**o):
    a = dict(pool=A, fmt=0, n_layers=1, n_pages=4, n_kv_heads=8, bt=A, bt_stride=4, slot=A, t0=A, n_tok=A, row0=A, M=1,
             max_tokens=16, total_rows=16, out_type=1, k_out=A, v_out=A)
    a.update(o)
    fa_dec.op_kv8_gather(**a)


def decode(**o):
    a = dict(q=A, M=1, n_heads=16, n_kv_heads=8, pos=A, slot=A, bt=A, bt_stride=4, n_pages=4, fmt=0, pool=A, scratch=A,
             scratch_bytes=1 << 40, out32=A)
    a.update(o)
    fa_dec.op_paged_attention_kv8(**a)


def prefill(**o):
    a = dict(q=A, M=1, n_heads=16, n_kv_heads=8, pos=A, slot=A, bt=A, bt_stride=4, n_pages=4, fmt=0, pool=A, tiles=A,
             n_tiles=1, scratch=A, scratch_bytes=1 << 40, out32=A)
    a.update(o)
    fa_dec.op_prefill_attention_kv8(**a)


CASES = (
    [(append, {n: 0}) for n in ("k", "v", "M", "n_layers", "n_kv_heads", "pos", "slot", "bt", "bt_stride", "n_pages",
                                "pool")]
    + [(append, o) for o in (dict(src_type=8), dict(fmt=2), dict(fmt=-1), dict(row_stride=1023), dict(row_stride=1028),
                             dict(row_stride=896), dict(k=A + 8), dict(v=A + 2), dict(pool=A + 64), dict(M=-3))]
    + [(qkv_append, {n: 0}) for n in ("qkv", "M", "n_heads", "n_kv_heads", "pos", "slot", "bt", "bt_stride", "n_pages",
                                      "qn", "kn", "rope", "max_pos", "pool", "q_out")]
    + [(qkv_append, o) for o in (dict(fmt=7), dict(qkv=A + 4), dict(pool=A + 16), dict(q_out=A + 8))]
    + [(gather, {n: 0}) for n in ("pool", "n_layers", "n_pages", "n_kv_heads", "bt", "bt_stride", "slot", "n_tok",
                                  "row0", "M", "max_tokens", "total_rows", "k_out", "v_out")]
    + [(gather, o) for o in (dict(fmt=2), dict(out_type=8), dict(M=65536), dict(n_layers=65536), dict(k_out=A + 8),
                             dict(v_out=A + 4), dict(pool=A + 32))]
    + [(f, {n: 0}) for f in (decode, prefill) for n in ("q", "M", "n_heads", "n_kv_heads", "pos", "slot", "bt",
                                                        "bt_stride", "n_pages", "pool", "out32")]
    + [(f, o) for f in (decode, prefill) for o in (
        dict(fmt=2), dict(n_heads=12), dict(n_heads=72), dict(n_heads=4), dict(q=A + 4), dict(pool=A + 64),
        dict(out32=A + 8), dict(out32=0, out16=A + 2), dict(out16_lo=A), dict(scratch=A + 8))]
    + [(prefill, o) for o in (dict(tiles=0), dict(n_tiles=0), dict(tiles=A + 4))]
)


@pytest.mark.parametrize("call,over", CASES, ids=lambda x: x.__name__ if callable(x) else "-".join(map(str, x)))
def test_bad_arguments_are_refused_on_the_host(call, over):
    with pytest.raises(fa_dec.FaError) as e:
        call(**over)
    assert e.value.code == INVALID
    assert str(e.value).split(": ")[1].startswith("fa_op_")


@pytest.mark.parametrize("call,over", [(append, dict(M=2 ** 31 - 1, n_layers=1000, row_stride=1024000)),
                                       (qkv_append, dict(n_heads=2 ** 16)),
                                       (gather, dict(bt_stride=2 ** 28)), (decode, dict(bt_stride=2 ** 28))],
                         ids=["append", "qkv_append", "gather", "decode"])
def test_sizes_past_the_kernels_range_are_refused(call, over):
    with pytest.raises(fa_dec.FaError) as e:
        call(**over)
    assert e.value.code == CAPACITY


def test_short_scratch_is_refused():
    need = fa_dec.op_attention_kv8_scratch_bytes(3, 16, 8)
    assert need > 0
    for o in (dict(scratch=0), dict(scratch_bytes=need - 1)):
        with pytest.raises(fa_dec.FaError) as e:
            decode(M=3, **o)
        assert e.value.code == INVALID and str(need) in str(e.value)
    need = fa_dec.op_prefill_attention_kv8_scratch_bytes(3, 16, 8)
    if need:
        with pytest.raises(fa_dec.FaError):
            prefill(n_tiles=3, scratch_bytes=need - 1)


def test_sizes_of_pages_and_scratch():
    assert [fa_dec.op_kv8_page_bytes(n) for n in (-1, 0, 1, 8)] == [0, 0, 4224, 8 * 4224]
    assert fa_dec.KV8_TILE_BYTES == P.TILE and fa_dec.KV8_TILE_BYTES % 128 == 0
    assert fa_dec.op_attention_kv8_scratch_bytes(0, 16, 8) == 0
    assert fa_dec.op_prefill_attention_kv8_scratch_bytes(0, 16, 8) == 0


def test_plain_quantiser_stays_within_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((500, 128)) * np.exp(rng.uniform(-30, 30, (500, 1)))).astype(np.float32)
    for fmt in (P.INT8, P.E4M3):
        q, d = P.quantise(x, fmt)
        y = P.values(q, fmt) * d[:, None].astype(np.float64)
        # int8: half a step of d; e4m3: 2^-4 of the value, or half of its smallest step 2^-9 d
        half = d[:, None] * 0.5 if fmt == P.INT8 else np.maximum(np.abs(x) * 2.0 ** -4, d[:, None] * 2.0 ** -10)
        assert (np.abs(y - x) <= half * (1 + 1e-12)).all()
        assert np.abs(P.values(q, fmt)).max(-1).min() > (126 if fmt == P.INT8 else 223)
        q0, d0 = P.quantise(np.zeros((1, 128), np.float32), fmt)
        assert not q0.any() and d0[0] == P.TINY


def test_plain_quantiser_ties_and_bad_values():
    x = np.zeros((2, 128), np.float32)
    x[0, :6] = [127, 0.5, 1.5, 2.5, -0.5, -1.5]                  # d = 1
    x[1, :3] = [np.inf, 1, np.nan]
    q, d = P.quantise(x, P.INT8)
    assert d[0] == 1 and q.view(np.int8)[0, :6].tolist() == [127, 0, 2, 2, 0, -2]
    assert np.isnan(d[1]) and not q[1].any()
    x[0, :6] = [448, 17, 19, 2.0 ** -10, 3 * 2.0 ** -10, -17]    # d = 1, step 2 at 16, 2^-9 at 0
    q, d = P.quantise(x, P.E4M3)
    assert d[0] == 1 and P.E4M3_VALUES[q[0, :6]].tolist() == [448, 16, 20, 0, 2.0 ** -8, -16]
    assert np.isnan(d[1]) and not q[1].any()
    for top, want in ((448, 1), (449, 2), (224, 0.5), (225, 1)):
        x[0, 0] = top
        x[0, 1:] = 0
        assert P.quantise(x, P.E4M3)[1][0] == want
