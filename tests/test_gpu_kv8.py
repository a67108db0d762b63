"""The 8-bit cache on the GPU against tests/kv8_plain.py: byte identity for the writes,
one rounding for the reads, derived bounds for the attention."""
import numpy as np
import pytest

import fa_dec
import kv8_plain as P
import oracle
from helpers import dev, rel_rms

pytestmark = pytest.mark.gpu

FORMATS = [P.INT8, P.E4M3]
IDS = ["int8", "e4m3"]
F16_NAN = 0x7fff


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


def _err(torch):
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _src(torch, x, src_type):
    """x (f32) on the device in src_type, and the same values as f32."""
    t = dev(torch, x).to({P.F32: torch.float32, P.F16: torch.float16, P.BF16: torch.bfloat16}[src_type])
    return t, t.float().cpu().numpy()


def _vectors(rng, *shape):
    """Head vectors of different sizes with a few large channels."""
    x = rng.standard_normal((*shape, 128)) * np.exp(0.5 * rng.standard_normal((*shape, 1)))
    x[..., ::37] *= 4
    return x.astype(np.float32)


def _table(rng, lens, n_pages, stride=None):
    stride = stride or max(-(-max(lens) // 16), 1)
    pages = rng.permutation(n_pages)
    bt, used = np.zeros((len(lens), stride), np.int32), 0
    for i, n in enumerate(lens):
        need = -(-n // 16)
        bt[i, :need] = pages[used:used + need]
        used += need
    return bt


def _garbage_pool(rng, layers, n_pages, hkv):
    """Random bytes: among them e4m3 NaN, and scales that are NaN, infinite or huge."""
    pool = rng.integers(0, 256, (layers, n_pages, hkv, P.TILE), dtype=np.uint8)
    pool[:, ::2, :, -128:] = 0xff
    return pool


def _append(torch, k, v, src_type, row_stride, M, layers, hkv, pos, slot, bt, n_pages, fmt, pool, err):
    fa_dec.op_kv8_append(k.data_ptr(), v.data_ptr(), src_type, row_stride, M, layers, hkv, pos.data_ptr(),
                         slot.data_ptr(), bt.data_ptr(), bt.shape[1], n_pages, fmt, pool.data_ptr(), err.data_ptr(),
                         _stream(torch))


# ------------------------------------------------------------------ append --
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("src_type,layers,hkv,M", [(P.F16, 1, 8, 1), (P.F32, 3, 8, 77), (P.BF16, 2, 5, 33),
                                                   (P.F16, 28, 8, 3), (P.F32, 1, 1, 19), (P.F32, 1, 64, 5)])
def test_append_bytes_are_exact(torch_cuda, fmt, src_type, layers, hkv, M):
    torch = torch_cuda
    rng = np.random.default_rng(M)
    lens = [M + 16, 40]
    n_pages = 2 * (-(-(M + 16) // 16) + 3) + 1
    bt = _table(rng, lens, n_pages)
    slot = np.where(np.arange(M) % 3 == 2, 1, 0).astype(np.int32)
    pos = np.where(slot == 1, np.arange(M) // 3, np.arange(M) + 7).astype(np.int32)
    pos[np.arange(M) % 5 == 4] = -1                              # padding rows
    order = rng.permutation(M)
    slot, pos = slot[order], pos[order]
    keep = (pos < 0) | (pos < np.where(slot == 1, 40, M + 16))
    pos[~keep] = -1
    # K and V as slices of one projection row with a gap behind them
    ld = 2 * layers * hkv * 128 + 64
    x = np.zeros((M, ld), np.float32)
    kv = _vectors(rng, 2, M, layers, hkv)
    kv[0, 0, 0, 0] = 0                                           # a zero vector
    kv[1, M // 2, -1, -1, 5] = 1000
    n = layers * hkv * 128
    x[:, :n], x[:, n:2 * n] = kv[0].reshape(M, n), kv[1].reshape(M, n)
    d_x, x = _src(torch, x, src_type)
    k, v = (x[:, i * n:(i + 1) * n].reshape(M, layers, hkv, 128) for i in (0, 1))
    pool = _garbage_pool(rng, layers, n_pages, hkv)
    d_pool, d_err = dev(torch, pool), _err(torch)
    _append(torch, d_x, d_x[:, n:], src_type, ld, M, layers, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt),
            n_pages, fmt, d_pool, d_err)
    slot_of = np.where(pos < 0, 0, slot)
    P.write(pool, bt, slot_of, pos, k, v, fmt)
    assert np.array_equal(d_pool.cpu().numpy(), pool)
    assert int(d_err) == 0


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_append_edge_vectors(torch_cuda, fmt):
    """Ties, the smallest and the largest f32, subnormals, infinities and NaN."""
    torch = torch_cuda
    rng = np.random.default_rng(5)
    M = 64
    x = _vectors(rng, 2, M, 1, 1)
    for i, scale in enumerate([1e-38, 1e-41, 1e-45, 1e30, 2e37, 1.0]):
        x[0, i] *= np.float32(scale)
    ties = (np.arange(128) - 64 + 0.5).astype(np.float32)
    ties[0] = 127
    x[0, 8, 0, 0] = ties                                          # d = 1 in int8: all ties
    x[0, 9, 0, 0] = ties * np.float32(1.7)                        # near ties of a rounded d
    x[0, 10, 0, 0] = np.where(np.arange(128) % 2, 1, -1) * np.float32(448 * 2.0 ** -5)
    x[0, 11, 0, 0] = np.concatenate([[448], np.arange(127) + 0.5]).astype(np.float32)
    x[0, 12, 0, 0, 7], x[0, 13, 0, 0, 127], x[0, 14, 0, 0, 0] = np.nan, np.inf, -np.inf
    x[0, 15] = np.finfo(np.float32).max
    x[0, 16] = 0
    x[0, 17] = -0.0
    # quotients next to a border: the neighbours of (k + 1/2) d for random d
    for m in range(20, M):
        amax = np.float32(rng.uniform(1, 2) * 2.0 ** rng.integers(-20, 20))
        d = np.float32(np.float64(amax) / 127)
        border = ((rng.integers(0, 127, 127) + 0.5) * np.float64(d)).astype(np.float32)
        step = rng.integers(-1, 2, 127)
        near = np.where(step < 0, np.nextafter(border, 0), np.where(step > 0, np.nextafter(border, np.inf), border))
        x[:, m, 0, 0] = np.concatenate([[amax], np.minimum(near.astype(np.float32), amax)])
    pos = np.arange(M, dtype=np.int32)
    bt = np.arange(4, dtype=np.int32)[None]
    pool = np.zeros((1, 4, 1, P.TILE), np.uint8)
    d_pool, d_err = dev(torch, pool), _err(torch)
    _append(torch, dev(torch, x[0]), dev(torch, x[1]), P.F32, 128, M, 1, 1, dev(torch, pos),
            dev(torch, np.zeros(M, np.int32)), dev(torch, bt), 4, fmt, d_pool, d_err)
    P.write(pool, bt, np.zeros(M, np.int32), pos, x[0], x[1], fmt)
    got, want = d_pool.cpu().numpy(), pool
    (q, d), (qw, dw) = P.parts(got), P.parts(want)
    assert np.array_equal(np.isnan(d), np.isnan(dw)) and np.array_equal(d[~np.isnan(d)], dw[~np.isnan(dw)])
    assert np.array_equal(q, qw)


@pytest.mark.parametrize("bad", ["pos", "past_table", "page", "page_negative", "slot"])
def test_append_flags_bad_rows_and_writes_the_others(torch_cuda, bad):
    torch = torch_cuda
    rng = np.random.default_rng(6)
    M, hkv, n_pages = 6, 8, 8
    k, v = _vectors(rng, M, 1, hkv), _vectors(rng, M, 1, hkv)
    bt = np.arange(8, dtype=np.int32).reshape(2, 4)[:, ::-1].copy()
    slot, pos = np.array([0, 0, 1, 1, 0, 1], np.int32), np.array([0, 17, 33, 5, 40, 63], np.int32)
    kb, want = bt.copy(), pos.copy()
    if bad == "pos": pos[2] = -2
    elif bad == "past_table": pos[2] = 64
    elif bad == "page": kb[1, 2] = n_pages
    elif bad == "page_negative": kb[1, 2] = -1
    else: slot[2] = -1
    want[2] = -1
    pool = _garbage_pool(rng, 1, n_pages, hkv)
    d_pool, d_err = dev(torch, pool), _err(torch)
    _append(torch, dev(torch, k), dev(torch, v), P.F32, 1024, M, 1, hkv, dev(torch, pos), dev(torch, slot),
            dev(torch, kb), n_pages, P.INT8, d_pool, d_err)
    P.write(pool, bt, np.maximum(slot, 0), want, k, v, P.INT8)
    assert np.array_equal(d_pool.cpu().numpy(), pool)
    assert int(d_err) == (2 if bad.startswith("page") else 4)


def test_append_reaches_pages_behind_2_gib(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(7)
    hkv, n_pages = 8, 70000                                       # 2.4 GB
    pool = torch.zeros((1, n_pages, hkv, P.TILE), dtype=torch.uint8, device="cuda")
    bt = np.array([[69999, 3, 65000]], np.int32)
    M = 48
    k, v = _vectors(rng, M, 1, hkv), _vectors(rng, M, 1, hkv)
    pos, slot, d_err = np.arange(M, dtype=np.int32), np.zeros(M, np.int32), _err(torch)
    d = [dev(torch, a) for a in (k, v, pos, slot, bt)]
    _append(torch, d[0], d[1], P.F32, 1024, M, 1, hkv, d[2], d[3], d[4], n_pages, P.INT8, pool, d_err)
    small = np.zeros((1, 3, hkv, P.TILE), np.uint8)
    P.write(small, np.array([[0, 1, 2]]), slot, pos, k, v, P.INT8)
    assert np.array_equal(pool[:, bt[0].tolist()].cpu().numpy(), small)
    q = dev(torch, (rng.standard_normal((1, 16, 128)) * 0.1).astype(np.float32))
    out = _decode(torch, q, 16, hkv, dev(torch, np.array([47], np.int32)), d[3][:1], d[4], n_pages, P.INT8, pool, d_err)
    want = P.attention(q.cpu().numpy()[0], *[x[0] for x in P.read(small, np.array([0, 1, 2]), 0, 48, P.INT8)])
    assert rel_rms(out.cpu().numpy()[0], want.reshape(-1)) < 5e-6
    assert int(d_err) == 0


# ------------------------------------------------------------ kernel 1 form --
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,M", [(16, 8, 1), (16, 8, 130), (5, 5, 17), (12, 4, 9), (16, 2, 33), (1, 1, 3)])
def test_qknorm_rope_append_matches_definition(torch_cuda, fmt, hq, hkv, M):
    torch = torch_cuda
    rng = np.random.default_rng(hq * 100 + M)
    max_pos, n_pages = 512, 40
    qkv = _vectors(rng, M, hq + 2 * hkv) * 2
    qkv[0, hq] = 0
    qn, kn = (rng.uniform(0.8, 1.2, 128).astype(np.float32) for _ in range(2))
    rope = np.asarray(oracle.rope_table(max_pos), np.float32).reshape(max_pos, 64, 2)
    bt = _table(rng, [max_pos], n_pages)
    pos = rng.permutation(max_pos)[:M].astype(np.int32)
    if M > 2:
        pos[1] = -1
    slot = np.where(pos < 0, 10 ** 6, 0).astype(np.int32)         # a padding row's slot is not looked at
    pool = _garbage_pool(rng, 1, n_pages, hkv)
    d_pool, d_err = dev(torch, pool), _err(torch)
    q_out = torch.full((M, hq, 128), 7.0, device="cuda")
    d = [dev(torch, a) for a in (qkv, pos, slot, bt, qn, kn, rope)]
    fa_dec.op_qknorm_rope_append_kv8(d[0].data_ptr(), M, hq, hkv, d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(),
                                     bt.shape[1], n_pages, d[4].data_ptr(), d[5].data_ptr(), 1e-5, d[6].data_ptr(),
                                     max_pos, fmt, d_pool.data_ptr(), q_out.data_ptr(), d_err.data_ptr(),
                                     _stream(torch))
    live = pos >= 0
    rot = rope[np.maximum(pos, 0)]
    q = P.norm_rotate(qkv[:, :hq], qn, rot) * np.float32(1 / np.sqrt(np.float32(128)))
    q[~live] = 7
    k = P.norm_rotate_exact(qkv[:, hq:hq + hkv], kn, rot)
    P.write(pool, bt, np.zeros(M, np.int32), pos, k[:, None], qkv[:, hq + hkv:][:, None], fmt)
    assert np.array_equal(q_out.cpu().numpy(), q)
    got = d_pool.cpu().numpy()
    (raw, d), (raw_w, d_w) = P.parts(got), P.parts(pool)
    # K's bytes are those of 64 bits; its int8 scale comes from the f32 maximum, which is off by
    # 2^-20 at most (an e4m3 scale is a power of two); V is exact
    assert np.array_equal(raw, raw_w)
    assert np.array_equal(d[..., 1, :].view(np.uint32), d_w[..., 1, :].view(np.uint32))
    live_d = np.isfinite(d_w[..., 0, :])
    assert np.array_equal(live_d, np.isfinite(d[..., 0, :]))
    off = np.abs(d[..., 0, :][live_d].astype(np.float64) - d_w[..., 0, :][live_d])
    assert (off <= np.abs(d_w[..., 0, :][live_d]) * (2.0 ** -20 if fmt == P.INT8 else 0)).all()
    assert int(d_err) == 0


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_qknorm_rope_append_keys_next_to_borders(torch_cuda, fmt):
    """A hundred thousand key vectors: every byte that of the 64-bit value rounded once, those
    within the f32 error of a border among them."""
    torch = torch_cuda
    rng = np.random.default_rng(23)
    hq, hkv, M, max_pos = 1, 40, 2500, 2512
    qkv = _vectors(rng, M, hq + 2 * hkv)
    w = np.ones(128, np.float32)
    rope = np.asarray(oracle.rope_table(max_pos), np.float32).reshape(max_pos, 64, 2)
    pos, n_pages = np.arange(M, dtype=np.int32), max_pos // 16
    bt = rng.permutation(n_pages).astype(np.int32)[None]
    pool, err = torch.zeros((1, n_pages, hkv, P.TILE), dtype=torch.uint8, device="cuda"), _err(torch)
    q = torch.zeros((M, hq, 128), device="cuda")
    d = [dev(torch, a) for a in (qkv, pos, np.zeros(M, np.int32), bt, w, rope)]
    p = [x.data_ptr() for x in d]
    fa_dec.op_qknorm_rope_append_kv8(p[0], M, hq, hkv, p[1], p[2], p[3], n_pages, n_pages, p[4], p[4], 1e-5, p[5],
                                     max_pos, fmt, pool.data_ptr(), q.data_ptr(), err.data_ptr(), _stream(torch))
    raw, _ = P.parts(pool.cpu().numpy())
    got = raw[0, bt[0, pos // 16], :, 0, pos % 16]
    want, _ = P.quantise(P.norm_rotate_exact(qkv[:, hq:hq + hkv], w, rope[:M]), fmt)
    assert np.array_equal(got, want) and int(err) == 0


def test_qknorm_rope_append_q_equals_the_f16_pools_op(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(21)
    M, max_pos = 37, 256
    qkv, pos = _vectors(rng, M, 32), rng.permutation(max_pos)[:M].astype(np.int32)
    d = [dev(torch, a) for a in (qkv, pos, np.zeros(M, np.int32), np.arange(16, dtype=np.int32)[None],
                                 np.ones(128, np.float32), np.ones(128, np.float32),
                                 np.asarray(oracle.rope_table(max_pos), np.float32))]
    p = [x.data_ptr() for x in d]
    q16, q8 = (torch.zeros((M, 16, 128), device="cuda") for _ in range(2))
    pool16 = torch.zeros((16, 8 * 2 * 16 * 128), dtype=torch.int16, device="cuda")
    pool8 = torch.zeros((16, 8, P.TILE), dtype=torch.uint8, device="cuda")
    err = _err(torch)
    fa_dec.op_qknorm_rope_append(p[0], M, p[1], p[2], p[3], 16, 16, p[4], p[5], 1e-5, p[6], max_pos, pool16.data_ptr(),
                                 q16.data_ptr(), err.data_ptr(), _stream(torch))
    fa_dec.op_qknorm_rope_append_kv8(p[0], M, 16, 8, p[1], p[2], p[3], 16, 16, p[4], p[5], 1e-5, p[6], max_pos, P.INT8,
                                     pool8.data_ptr(), q8.data_ptr(), err.data_ptr(), _stream(torch))
    assert torch.equal(q16, q8)
    # the f16 cache rounds a value by 2^-11 of it at most, the 8-bit one by half a step
    f16 = pool16.view(torch.float16).reshape(16, 8, 2, 16, 128).float().cpu().numpy()
    raw, d8 = P.parts(pool8.cpu().numpy())
    off = np.abs(P.values(raw, P.INT8) * d8[..., None] - f16)
    assert (off <= d8[..., None] * 0.5 * (1 + 1e-6) + np.abs(f16) * 2.0 ** -11).all()
    assert int(err) == 0


def test_qknorm_rope_append_flags_bad_rows(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(22)
    for pos, page, bits in ((-2, 0, 4), (64, 0, 4), (40, 0, 4), (3, 9, 2), (3, -1, 2)):
        d = [dev(torch, a) for a in (_vectors(rng, 1, 32), np.array([pos], np.int32), np.zeros(1, np.int32),
                                     np.array([[page, 1]], np.int32), np.ones(128, np.float32),
                                     np.asarray(oracle.rope_table(64), np.float32))]
        p = [x.data_ptr() for x in d]
        q, err = torch.zeros((1, 16, 128), device="cuda"), _err(torch)
        pool = torch.full((4, 8, P.TILE), 77, dtype=torch.uint8, device="cuda")
        fa_dec.op_qknorm_rope_append_kv8(p[0], 1, 16, 8, p[1], p[2], p[3], 2, 4, p[4], p[4], 1e-5, p[5], 64, P.INT8,
                                         pool.data_ptr(), q.data_ptr(), err.data_ptr(), _stream(torch))
        assert int(err) == bits and bool((pool == 77).all())


# ------------------------------------------------------------------ gather --
def _filled(rng, lens, layers, hkv, fmt, n_pages=None, spread=0.5):
    """A pool of garbage with these sequences written into it, the table and the read-back."""
    n_pages = n_pages or sum(-(-n // 16) for n in lens) + 3
    bt = _table(rng, lens, n_pages)
    pool = _garbage_pool(rng, layers, n_pages, hkv)
    raw, scales = P.parts(pool)
    for i, n in enumerate(lens):
        if not n:
            continue
        x = rng.standard_normal((2, n, layers, hkv, 128)) * np.exp(spread * rng.standard_normal((2, n, layers, hkv, 1)))
        q, d = P.quantise(x.astype(np.float32), fmt)
        t = np.arange(n)
        for part in (0, 1):
            raw[:, bt[i, t // 16], :, part, t % 16] = q[part]
            scales[:, bt[i, t // 16], :, part, t % 16] = d[part]
    return pool, bt, n_pages


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("out_type,layers,hkv", [(P.F16, 3, 8), (P.BF16, 1, 5), (P.F32, 2, 1), (P.F16, 1, 11)])
def test_gather_ragged_ranges(torch_cuda, fmt, out_type, layers, hkv):
    torch = torch_cuda
    rng = np.random.default_rng(hkv)
    lens = [1, 16, 17, 320, 47, 33, 5]
    pool, bt, n_pages = _filled(rng, lens, layers, hkv, fmt)
    t0 = np.array([0, 0, 16, 3, 31, 0, 2], np.int32)
    n_tok = np.array([1, 16, 1, 301, 2, 0, 3], np.int32)
    slot = np.arange(7, dtype=np.int32)
    order = rng.permutation(7)
    row0 = np.zeros(7, np.int32)
    at = 2
    for m in order:
        row0[m] = at
        at += n_tok[m] + 1                                        # gaps
    total = at + 3
    dt = {P.F32: torch.float32, P.F16: torch.float16, P.BF16: torch.bfloat16}[out_type]
    k_out, v_out = (torch.full((layers, hkv, total, 128), 9.0, dtype=dt, device="cuda") for _ in range(2))
    d = [dev(torch, a) for a in (pool, bt, slot[order], t0[order], n_tok[order], row0[order])]
    p, err = [x.data_ptr() for x in d], _err(torch)
    fa_dec.op_kv8_gather(p[0], fmt, layers, n_pages, hkv, p[1], bt.shape[1], p[2], p[3], p[4], p[5], 7, 301, total,
                         out_type, k_out.data_ptr(), v_out.data_ptr(), err.data_ptr(), _stream(torch))
    want = np.full((2, layers, hkv, total, 128), 9.0)
    for m in range(7):
        kv = P.read(pool, bt[m], t0[m], t0[m] + n_tok[m], fmt)
        for part in (0, 1):
            want[part, :, :, row0[m]:row0[m] + n_tok[m]] = kv[part]
    for part, got in ((0, k_out), (1, v_out)):
        # d q is formed in f32 and rounded to the type: the f32 product of the definition, rounded once
        w = torch.from_numpy(want[part].astype(np.float32)).to(dt)
        assert torch.equal(got.cpu(), w)
    assert int(err) == 0
    if not t0[0]:                                                 # NULL t0: from the first token
        one = torch.zeros((layers, hkv, 1, 128), dtype=dt, device="cuda")
        two = torch.zeros_like(one)
        z = dev(torch, np.zeros(1, np.int32))
        fa_dec.op_kv8_gather(p[0], fmt, layers, n_pages, hkv, p[1], bt.shape[1], z.data_ptr(), 0,
                             dev(torch, np.ones(1, np.int32)).data_ptr(), z.data_ptr(), 1, 1, 1, out_type,
                             one.data_ptr(), two.data_ptr(), err.data_ptr(), _stream(torch))
        assert torch.equal(one.cpu(), torch.from_numpy(want[0][:, :, row0[0]:row0[0] + 1].astype(np.float32)).to(dt))


@pytest.mark.parametrize("over,bits", [(dict(n_tok=17), 8), (dict(n_tok=-1), 8), (dict(t0=-1), 8), (dict(t0=20), 8),
                                       (dict(row0=-1), 8), (dict(row0=17), 8), (dict(slot=-1), 8),
                                       (dict(page=3), 2), (dict(page=-1), 2), (dict(t0=2 ** 31 - 8), 8),
                                       (dict(row0=2 ** 31 - 1), 8)], ids=str)
def test_gather_flags_bad_ranges(torch_cuda, over, bits):
    torch = torch_cuda
    a = dict(slot=0, t0=0, n_tok=16, row0=0, page=1)
    a.update(over)
    pool = torch.zeros((1, 3, 8, P.TILE), dtype=torch.uint8, device="cuda")
    d = {k: dev(torch, np.array([a[k]], np.int32)) for k in ("slot", "t0", "n_tok", "row0")}
    bt = dev(torch, np.array([[a["page"], 2]], np.int32))
    k_out, v_out = (torch.full((1, 8, 32, 128), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    err = _err(torch)
    fa_dec.op_kv8_gather(pool.data_ptr(), P.INT8, 1, 3, 8, bt.data_ptr(), 2, d["slot"].data_ptr(), d["t0"].data_ptr(),
                         d["n_tok"].data_ptr(), d["row0"].data_ptr(), 1, 16, 32, P.F16, k_out.data_ptr(),
                         v_out.data_ptr(), err.data_ptr(), _stream(torch))
    assert int(err) == bits
    assert bool((k_out == 9).all()) and bool((v_out == 9).all())


# --------------------------------------------------------------- attention --
def _scratch(torch, size):
    return torch.full((max(size, 16),), 0xff, dtype=torch.uint8, device="cuda")      # NaN bytes: nothing is read unwritten


def _decode(torch, q, hq, hkv, pos, slot, bt, n_pages, fmt, pool, err, out16=None, out16_lo=None, out=None):
    M = q.shape[0]
    out = torch.full((M, hq * 128), 5.0, device="cuda") if out is None else out
    size = fa_dec.op_attention_kv8_scratch_bytes(M, hq, hkv)
    scratch = _scratch(torch, size)
    fa_dec.op_paged_attention_kv8(q.data_ptr(), M, hq, hkv, pos.data_ptr(), slot.data_ptr(), bt.data_ptr(),
                                  bt.shape[1], n_pages, fmt, pool.data_ptr(), scratch.data_ptr(), size,
                                  out32=out.data_ptr(), err=err.data_ptr(), stream=_stream(torch),
                                  out16=0 if out16 is None else out16.data_ptr(),
                                  out16_lo=0 if out16_lo is None else out16_lo.data_ptr())
    return out


def _tiles(rows, step):
    """(first row, rows) pairs covering runs of rows (first, count)."""
    return np.array([(f + i, min(step, n - i)) for f, n in rows for i in range(0, n, step)], np.int32)


def _prefill(torch, q, hq, hkv, pos, slot, bt, n_pages, fmt, pool, tiles, err, out16=None, out16_lo=None, out=None):
    M = q.shape[0]
    out = torch.full((M, hq * 128), 5.0, device="cuda") if out is None else out
    size = fa_dec.op_prefill_attention_kv8_scratch_bytes(len(tiles), hq, hkv)
    scratch, d_tiles = _scratch(torch, size), dev(torch, tiles)
    fa_dec.op_prefill_attention_kv8(q.data_ptr(), M, hq, hkv, pos.data_ptr(), slot.data_ptr(), bt.data_ptr(),
                                    bt.shape[1], n_pages, fmt, pool.data_ptr(), d_tiles.data_ptr(), len(tiles),
                                    scratch.data_ptr(), size, out32=out.data_ptr(), err=err.data_ptr(),
                                    stream=_stream(torch), out16=0 if out16 is None else out16.data_ptr(),
                                    out16_lo=0 if out16_lo is None else out16_lo.data_ptr())
    return out


def _bound(q, k, v):
    """Largest error of an output of a row: a score is off by 2^-18 of sum |q k| at most (f32
    sums of 128 products that carry 22 bits: 128 x 2^-24 + 2^-22 < 2^-16.9 if every rounding
    went the same way, 2^-20 as they fall; an eighth of the former), a weight by that times ln 2
    relative, and the weighted sum by 2^-18 of the largest |v|."""
    g = len(q) // len(k)
    s = max(float((np.abs(k[h // g]) @ np.abs(q[h].astype(np.float64))).max()) for h in range(len(q)))
    return 2 * (2.0 ** -18 * s + 2.0 ** -18) * float(np.abs(v).max())


LENS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 255, 256, 257, 640, 1000]


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 8), (12, 4), (16, 2), (32, 8), (5, 5), (5, 1), (1, 1), (7, 1)])
def test_decode_attention_ragged(torch_cuda, fmt, hq, hkv):
    torch = torch_cuda
    rng = np.random.default_rng(hq * 10 + hkv)
    pool, bt, n_pages = _filled(rng, LENS, 1, hkv, fmt)
    order = rng.permutation(len(LENS))
    slot = np.concatenate([order, [10 ** 6, 3]]).astype(np.int32)
    pos = np.array([LENS[i] - 1 for i in order] + [-1, 4], np.int32)      # a padding row; a second row of sequence 3
    M = len(slot)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    out16, lo = (torch.zeros((M, hq * 128), dtype=torch.float16, device="cuda") for _ in range(2))
    got = _decode(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
                  dev(torch, pool), err, out16, lo)
    o32, pair = got.cpu().numpy(), (out16.float() + lo.float()).cpu().numpy()
    assert int(err) == 0
    for m in range(M):
        if pos[m] < 0:
            assert not o32[m].any() and not pair[m].any()
            continue
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, fmt))
        want = P.attention(q[m], k, v).reshape(-1)
        assert np.abs(o32[m] - want).max() <= _bound(q[m], k, v)
        assert rel_rms(o32[m], want) <= 5e-6, (m, pos[m])
        # the pair keeps 22 bits of the f32 output, its low part down to the f16 subnormals
        assert np.abs(pair[m] - o32[m]).max() <= np.abs(o32[m]).max() * 2.0 ** -21 + 2.0 ** -24
    assert np.array_equal(out16.cpu().numpy(), got.cpu().numpy().astype(np.float16))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n,hq,hkv,M", [(4001, 16, 8, 1), (20000, 16, 8, 2), (40960, 8, 1, 1), (9999, 32, 4, 3)])
def test_decode_attention_long(torch_cuda, fmt, n, hq, hkv, M):
    torch = torch_cuda
    rng = np.random.default_rng(n)
    lens = [n - 37 * i for i in range(M)]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, fmt)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _decode(torch, dev(torch, q), hq, hkv, dev(torch, np.array(lens, np.int32) - 1),
                  dev(torch, np.arange(M, dtype=np.int32)), dev(torch, bt), n_pages, fmt, dev(torch, pool), err)
    for m in range(M):
        k, v = (x[0] for x in P.read(pool, bt[m], 0, lens[m], fmt))
        want = P.attention(q[m], k, v).reshape(-1)
        assert rel_rms(got[m].cpu().numpy(), want) <= 5e-6
    assert int(err) == 0


@pytest.mark.parametrize("kind", ["sharp", "scales", "q_small", "q_large", "zeros"])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_attention_value_ranges(torch_cuda, fmt, which, kind):
    """Scores far apart, vectors whose sizes differ by many powers of ten, tiny and huge
    queries, zero vectors."""
    torch = torch_cuda
    rng = np.random.default_rng(3)
    hq, hkv, n, M = 16, 8, 300, 20
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    raw, scales = P.parts(pool)
    page, t = bt[0, np.arange(n) // 16], np.arange(n) % 16
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    if kind == "sharp":
        q *= 20
    elif kind == "scales":      # K and V sizes over many decades; the weight of a large V stays what it is
        scales[0, page, :, 0, t] *= (10.0 ** rng.uniform(-6, 0, (n, hkv))).astype(np.float32)
        scales[0, page, :, 1, t] *= (10.0 ** rng.uniform(-12, 12, (n, hkv))).astype(np.float32)
    elif kind == "q_small":
        q *= np.float32(1e-30)
    elif kind == "q_large":     # scores of thousands over keys of 1e-3
        q *= np.float32(1e6)
        scales[0, page, :, 0, t] *= np.float32(1e-4)
    else:
        raw[0, page[::3], :, 1, t[::3]] = 0
        scales[0, page[::3], :, 1, t[::3]] = P.TINY
        q[:, 3] = 0
    pos = np.arange(n - M, n).astype(np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = _decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)
    got = got.cpu().numpy().reshape(M, hq, 128)
    for m in range(M):
        k, v = (x[0] for x in P.read(pool, bt[0], 0, pos[m] + 1, fmt))
        want = P.attention(q[m], k, v)
        for h in range(hq):
            b = _bound(q[m, h:h + 1], k[h // 2:h // 2 + 1], v[h // 2:h // 2 + 1])
            assert np.abs(got[m, h] - want[h]).max() <= b, (m, h)
    assert int(err) == 0


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_nan_vectors_reach_their_own_rows_only(torch_cuda, fmt, which):
    """A token whose K or V vector is NaN makes the rows that see it NaN, on its head alone;
    rows before it, other sequences and masked places are untouched."""
    torch = torch_cuda
    rng = np.random.default_rng(4)
    hq, hkv, lens = 16, 8, [70, 70]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, fmt)
    _, scales = P.parts(pool)
    scales[0, bt[0, 50 // 16], 2, 0, 50 % 16] = np.nan            # K of token 50, KV head 2
    scales[0, bt[0, 60 // 16], 5, 1, 60 % 16] = np.nan            # V of token 60, KV head 5
    M = 140
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    pos, slot = np.tile(np.arange(70), 2).astype(np.int32), np.repeat([0, 1], 70).astype(np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
            dev(torch, pool))
    err = _err(torch)
    got = _decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, 70), (70, 70)], 64), err)
    nan = np.isnan(got.cpu().numpy().reshape(M, hq, 128))
    want = np.zeros_like(nan)
    want[50:70, 4:6] = True
    want[60:70, 10:12] = True
    assert np.array_equal(nan, want)


@pytest.mark.parametrize("step", [0.05, 0.4, 3.0, -0.05, -0.4, -3.0])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_scores_that_rise_or_fall_along_the_context(torch_cuda, fmt, which, step):
    """Score t is step * t of the row's largest length and a little noise: the running maximum
    rises by less and by more than what a kernel may leave it behind, or is the first score."""
    torch = torch_cuda
    rng = np.random.default_rng(17)
    hq, hkv, n, M = 16, 8, 333, 12
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    raw, scales = P.parts(pool)
    way = rng.choice([-1.0, 1.0], 128)
    t = np.arange(n)
    k = way * (step * t / 128)[:, None] + 0.002 * rng.standard_normal((hkv, n, 128)) * max(abs(step), 0.1)
    qk, dk = P.quantise(k.astype(np.float32), fmt)
    raw[0, bt[0, t // 16], :, 0, t % 16] = qk.transpose(1, 0, 2)
    scales[0, bt[0, t // 16], :, 0, t % 16] = dk.T
    q = (way + 0.01 * rng.standard_normal((M, hq, 128))).astype(np.float32)
    pos = np.arange(n - M, n).astype(np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = (_decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)).cpu().numpy()
    assert int(err) == 0
    for m in range(M):
        kk, v = (x[0] for x in P.read(pool, bt[0], 0, pos[m] + 1, fmt))
        assert np.abs(got[m] - P.attention(q[m], kk, v).reshape(-1)).max() <= _bound(q[m], kk, v), m


@pytest.mark.parametrize("base,M", [(0, 70), (37, 64), (500, 100), (1000, 20)])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_large_later_values_leave_earlier_rows(torch_cuda, fmt, which, base, M):
    """K and V of 1e30 in the second half of a chunk: a row before them is as accurate, in terms
    of what it attends to, as without them."""
    torch = torch_cuda
    rng = np.random.default_rng(base + M)
    hq, hkv, n = 16, 8, base + M
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    _, scales = P.parts(pool)
    late = np.arange(base + M // 2, n)
    for part in (0, 1):
        scales[0, bt[0, late // 16], :, part, late % 16] *= np.float32(1e30)
    pos = np.arange(base, n).astype(np.int32)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = (_decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)).cpu().numpy()
    assert int(err) == 0
    for m in range(M // 2):
        k, v = (x[0] for x in P.read(pool, bt[0], 0, pos[m] + 1, fmt))
        assert np.abs(got[m] - P.attention(q[m], k, v).reshape(-1)).max() <= _bound(q[m], k, v), m


@pytest.mark.parametrize("bad", ["pos", "past_table", "slot", "page", "page_negative"])
def test_decode_attention_flags_bad_rows(torch_cuda, bad):
    torch = torch_cuda
    rng = np.random.default_rng(8)
    hq, hkv, lens = 16, 8, [40, 200, 64]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, P.INT8)
    pos, slot = np.array([39, 199, 63], np.int32), np.array([0, 1, 2], np.int32)
    q = (rng.standard_normal((3, hq, 128)) * 0.3).astype(np.float32)
    kb = bt.copy()
    if bad == "pos": pos[1] = -2
    elif bad == "past_table": pos[1] = 16 * bt.shape[1]
    elif bad == "slot": slot[1] = -1
    elif bad == "page": kb[1, 3] = n_pages
    else: kb[1, 3] = -1
    err = _err(torch)
    got = _decode(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, kb), n_pages, P.INT8,
                  dev(torch, pool), err).cpu().numpy()
    assert int(err) == (2 if bad.startswith("page") else 8)
    for m in (0, 1, 2):
        k, v = (x[0] for x in P.read(pool, bt[m], 0, lens[m], P.INT8))
        if m == 1 and bad.startswith("page"):                     # the bad page's tokens are left out
            keep = np.r_[0:48, 64:200]
            k, v = k[:, keep], v[:, keep]
        elif m == 1:
            assert (got[1] == 5).all()
            continue
        assert rel_rms(got[m], P.attention(q[m], k, v).reshape(-1)) <= 5e-6


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,M,pages", [
    (16, 8, 1, 32), (16, 8, 1, 33), (16, 8, 8, 33), (16, 8, 9, 64), (16, 8, 9, 65), (16, 8, 18, 64), (16, 8, 19, 20),
    (16, 8, 55, 9), (16, 8, 56, 9), (32, 4, 30, 12), (32, 4, 50, 12), (7, 1, 100, 3), (1, 1, 3, 1)])
def test_decode_attention_table_widths(torch_cuda, fmt, hq, hkv, M, pages):
    """Rows of any length up to the table's, the longest among them, with padding rows, a bad slot
    and a bad page: on both sides of the sizes at which a call is cut into work another way."""
    torch = torch_cuda
    rng = np.random.default_rng(100 * pages + M)
    lens = rng.integers(1, 16 * pages + 1, M)
    lens[0] = 16 * pages
    pool, bt, n_pages = _filled(rng, lens.tolist(), 1, hkv, fmt)
    assert bt.shape[1] == pages
    pos, slot = (lens - 1).astype(np.int32), np.arange(M, dtype=np.int32)
    kb, left, missing = bt.copy(), {}, -1
    if M > 4:
        pos[2], slot[3] = -1, -5
        left = {2: 0.0, 3: 5.0}
        missing = int(np.argmax(lens[4:])) + 4                    # loses its first page
        kb[missing, 0] = n_pages + 7
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _decode(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, kb), n_pages, fmt,
                  dev(torch, pool), err).cpu().numpy()
    assert int(err) == (10 if M > 4 else 0)
    for m in range(M):
        if m in left:
            assert (got[m] == left[m]).all()
            continue
        k, v = (x[0] for x in P.read(pool, bt[m], 0, lens[m], fmt))
        if m == missing:
            k, v = k[:, 16:], v[:, 16:]
        want = P.attention(q[m], k, v).reshape(-1) if k.shape[1] else np.zeros(hq * 128)
        assert np.abs(got[m] - want).max() <= (_bound(q[m], k, v) if k.shape[1] else 0), m


# ----------------------------------------------------------------- prefill --
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,chunks", [
    (16, 8, [(0, 112)]), (16, 8, [(0, 1), (5, 1), (63, 2), (64, 65)]), (16, 8, [(700, 130), (0, 64), (15, 17)]),
    (8, 8, [(33, 200)]), (12, 4, [(100, 90)]), (16, 2, [(70, 40), (0, 16)]), (5, 1, [(20, 60)]), (32, 8, [(250, 70)]),
    (7, 1, [(3, 37)]), (1, 1, [(0, 129)])])
def test_prefill_attention_ragged(torch_cuda, fmt, hq, hkv, chunks):
    torch = torch_cuda
    rng = np.random.default_rng(len(chunks) * 100 + hq)
    lens = [b + n for b, n in chunks]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, fmt)
    pos = np.concatenate([np.arange(b, b + n) for b, n in chunks]).astype(np.int32)
    slot = np.repeat(np.arange(len(chunks)), [n for _, n in chunks]).astype(np.int32)
    first = np.concatenate([[0], np.cumsum([n for _, n in chunks])[:-1]])
    tiles = _tiles([(int(f), n) for f, (_, n) in zip(first, chunks)], 128 * hkv // hq)
    M = len(pos)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    out16, lo = (torch.zeros((M, hq * 128), dtype=torch.float16, device="cuda") for _ in range(2))
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
                   dev(torch, pool), tiles, err, out16, lo).cpu().numpy()
    pair = (out16.float() + lo.float()).cpu().numpy()
    assert int(err) == 0
    for m in range(M):
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, fmt))
        want = P.attention(q[m], k, v).reshape(-1)
        assert np.abs(got[m] - want).max() <= _bound(q[m], k, v)
        assert rel_rms(got[m], want) <= 5e-6, m
        assert np.abs(pair[m] - got[m]).max() <= np.abs(got[m]).max() * 2.0 ** -21 + 2.0 ** -24


def test_prefill_attention_repeated_and_padded_rows(torch_cuda):
    """Positions that repeat within a tile, rows of no tile, and a tile that begins with padding."""
    torch = torch_cuda
    rng = np.random.default_rng(9)
    hq, hkv = 16, 8
    pool, bt, n_pages = _filled(rng, [90], 1, hkv, P.INT8)
    pos = np.array([-1, -1, 40, 40, 41, 89, 89, 7], np.int32)
    M = len(pos)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt),
                   n_pages, P.INT8, dev(torch, pool), np.array([[0, 7]], np.int32), err).cpu().numpy()
    assert not got[:2].any() and (got[7] == 5).all() and int(err) == 0
    for m in range(2, 7):
        k, v = (x[0] for x in P.read(pool, bt[0], 0, pos[m] + 1, P.INT8))
        assert rel_rms(got[m], P.attention(q[m], k, v).reshape(-1)) <= 5e-6


@pytest.mark.parametrize("tile,pos,page,bits", [
    ((0, 0), None, None, 4), ((0, 65), None, None, 4), ((-1, 4), None, None, 4), ((70, 64), None, None, 4),
    ((2 ** 31 - 1, 4), None, None, 4), ((64, 64), -2, None, 8), ((64, 64), 10 ** 6, None, 8), ((64, 64), None, 99, 2),
    ((64, 64), None, -1, 2)])
def test_prefill_attention_flags_bad_tiles(torch_cuda, tile, pos, page, bits):
    """The tile beside the bad one is computed; a bad tile or row writes nothing."""
    torch = torch_cuda
    rng = np.random.default_rng(10)
    hq, hkv = 16, 8
    pool, bt, n_pages = _filled(rng, [128], 1, hkv, P.INT8)
    p = np.arange(128, dtype=np.int32)
    if pos is not None:
        p[127] = pos
    kb = bt.copy()
    if page is not None:
        kb[0, 5] = page                                           # tokens 80..95
    q = (rng.standard_normal((128, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, p), dev(torch, np.zeros(128, np.int32)), dev(torch, kb),
                   n_pages, P.INT8, dev(torch, pool), np.array([[0, 64], tile], np.int32), err).cpu().numpy()
    assert int(err) == bits
    if tile[0] != 0:
        k, v = (x[0] for x in P.read(pool, bt[0], 0, 128, P.INT8))
        for m in range(64):
            assert rel_rms(got[m], P.attention(q[m], k[:, :m + 1], v[:, :m + 1]).reshape(-1)) <= 5e-6
        if pos is not None:
            assert (got[127] == 5).all()
        if page is not None:                                      # the bad page's tokens are left out
            keep = np.r_[0:80, 96:128]
            assert rel_rms(got[127], P.attention(q[127], k[:, keep], v[:, keep]).reshape(-1)) <= 5e-6
        elif bits == 4:
            assert (got[64:] == 5).all()


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,chunks", [
    (16, 8, [(4000, 3)]), (16, 8, [(1100, 64), (3000, 70)]), (8, 1, [(6000, 20)]), (32, 8, [(2500, 32)]),
    (5, 5, [(1500, 130)]), (16, 2, [(9000, 1)])])
def test_prefill_attention_few_tiles_over_long_contexts(torch_cuda, fmt, hq, hkv, chunks):
    """Calls of few tiles, whose keys are cut into parts: every row against the definition."""
    torch = torch_cuda
    rng = np.random.default_rng(hq + chunks[0][0])
    lens = [b + n for b, n in chunks]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, fmt)
    pos = np.concatenate([np.arange(b, b + n) for b, n in chunks]).astype(np.int32)
    slot = np.repeat(np.arange(len(chunks)), [n for _, n in chunks]).astype(np.int32)
    first = np.concatenate([[0], np.cumsum([n for _, n in chunks])[:-1]])
    tiles = _tiles([(int(f), n) for f, (_, n) in zip(first, chunks)], 128 * hkv // hq)
    assert fa_dec.op_prefill_attention_kv8_scratch_bytes(len(tiles), hq, hkv) > 0
    M = len(pos)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    out16, lo = (torch.zeros((M, hq * 128), dtype=torch.float16, device="cuda") for _ in range(2))
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
                   dev(torch, pool), tiles, err, out16, lo).cpu().numpy()
    pair = (out16.float() + lo.float()).cpu().numpy()
    assert int(err) == 0
    for m in range(M):
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, fmt))
        want = P.attention(q[m], k, v).reshape(-1)
        assert np.abs(got[m] - want).max() <= _bound(q[m], k, v)
        assert rel_rms(got[m], want) <= 5e-6, m
        assert np.abs(pair[m] - got[m]).max() <= np.abs(got[m]).max() * 2.0 ** -21 + 2.0 ** -24


def test_prefill_attention_parts_with_padding_nan_and_a_bad_page(torch_cuda):
    """Keys in parts: rows that see none of a part's keys, a NaN vector in the last part only,
    a page outside the pool in the middle, a row of another sequence."""
    torch = torch_cuda
    rng = np.random.default_rng(14)
    hq, hkv, n = 16, 8, 4000
    pool, bt, n_pages = _filled(rng, [n, 64], 1, hkv, P.INT8)
    _, scales = P.parts(pool)
    scales[0, bt[0, 3900 // 16], 3, 1, 3900 % 16] = np.nan
    kb = bt.copy()
    kb[0, 2000 // 16] = n_pages + 7                               # tokens 2000..2015
    pos = np.array([-1, 5, 63, 1500, 3899, 3900, 3999, 3999], np.int32)
    slot = np.array([77, 0, 0, 0, 0, 0, 0, 1], np.int32)
    M = len(pos)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, kb), n_pages, P.INT8,
                   dev(torch, pool), np.array([[0, 8]], np.int32), err).cpu().numpy()
    assert int(err) == 2 | 8
    assert not got[0].any() and (got[7] == 5).all()
    for m in range(1, 7):
        keep = np.array([t for t in range(pos[m] + 1) if not 2000 <= t < 2016])
        k, v = (x[0][:, keep] for x in P.read(pool, bt[0], 0, pos[m] + 1, P.INT8))
        want, out = P.attention(q[m], k, v), got[m].reshape(hq, 128)
        heads = [h for h in range(hq) if not (pos[m] >= 3900 and h // 2 == 3)]
        assert rel_rms(out[heads], want[heads]) <= 5e-6, m
        assert np.isnan(out).all(-1).tolist() == [h not in heads for h in range(hq)]


@pytest.mark.parametrize("hq,hkv,M,longest", [(16, 8, 700, 40), (64, 64, 9, 300), (8, 2, 1500, 17), (200, 200, 3, 50),
                                               (16, 8, 2, 16)])
def test_decode_attention_many_short_rows_and_many_heads(torch_cuda, hq, hkv, M, longest):
    """More rows than a CTA has threads, rows of one page beside long ones, padding runs, more KV
    heads than usual; f16 output alone, no error word."""
    torch = torch_cuda
    rng = np.random.default_rng(M)
    lens = rng.integers(1, longest + 1, 40).tolist()
    lens[3] = 3 * longest
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, P.INT8)
    slot = rng.integers(0, 40, M).astype(np.int32)
    pos = np.array([rng.integers(0, lens[s]) for s in slot], np.int32)
    pos[M // 3:M // 3 + M // 5] = -1
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    out16 = torch.full((M, hq * 128), 5.0, dtype=torch.float16, device="cuda")
    size = fa_dec.op_attention_kv8_scratch_bytes(M, hq, hkv)
    d = [dev(torch, a) for a in (q, pos, slot, bt, pool)]
    p, scratch = [x.data_ptr() for x in d], _scratch(torch, size)
    fa_dec.op_paged_attention_kv8(p[0], M, hq, hkv, p[1], p[2], p[3], bt.shape[1], n_pages, P.INT8, p[4],
                                  scratch.data_ptr(), size, out16=out16.data_ptr(), stream=_stream(torch))
    got = out16.float().cpu().numpy()
    for m in np.unique(np.concatenate([np.arange(0, M, max(1, M // 60)), [M - 1]])):
        if pos[m] < 0:
            assert not got[m].any()
            continue
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, P.INT8))
        want = P.attention(q[m], k, v).reshape(-1)
        # half a step of f16 (2^-11 relative, 2^-25 among the subnormals) on top of the f32 bound
        assert (np.abs(got[m] - want) <= _bound(q[m], k, v) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()


def test_all_rows_padding(torch_cuda):
    torch = torch_cuda
    hq, hkv, M = 16, 8, 70
    pos, slot = dev(torch, np.full(M, -1, np.int32)), dev(torch, np.full(M, 10 ** 6, np.int32))
    bt, pool = dev(torch, np.full((1, 4), 99, np.int32)), torch.full((1, 2, hkv, P.TILE), 255, dtype=torch.uint8, device="cuda")
    q, err = torch.full((M, hq, 128), float("nan"), device="cuda"), _err(torch)
    assert not bool(_decode(torch, q, hq, hkv, pos, slot, bt, 2, P.E4M3, pool, err).any())
    assert not bool(_prefill(torch, q, hq, hkv, pos, slot, bt, 2, P.E4M3, pool, _tiles([(0, M)], 64), err).any())
    kv = torch.ones((M, hkv * 128), device="cuda")
    _append(torch, kv, kv, P.F32, hkv * 128, M, 1, hkv, pos, slot, bt, 2, P.E4M3, pool, err)
    assert bool((pool == 255).all()) and int(err) == 0


def test_prefill_from_a_graph_and_two_at_once(torch_cuda):
    """One captured prefill call (keys in parts) replayed with other positions, while another
    call with scratch of its own runs on a second stream."""
    torch = torch_cuda
    rng = np.random.default_rng(15)
    hq, hkv, n, M = 16, 8, 3000, 40
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, P.E4M3)
    d_pool, d_bt, slot = dev(torch, pool), dev(torch, bt), dev(torch, np.zeros(M, np.int32))
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    d_q, pos, err = dev(torch, q), dev(torch, np.arange(M, dtype=np.int32)), _err(torch)
    tiles = dev(torch, np.array([[0, M]], np.int32))
    size = fa_dec.op_prefill_attention_kv8_scratch_bytes(1, hq, hkv)
    scratch, out = _scratch(torch, size), torch.zeros((M, hq * 128), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fa_dec.op_prefill_attention_kv8(d_q.data_ptr(), M, hq, hkv, pos.data_ptr(), slot.data_ptr(), d_bt.data_ptr(),
                                        bt.shape[1], n_pages, P.E4M3, d_pool.data_ptr(), tiles.data_ptr(), 1,
                                        scratch.data_ptr(), size, out32=out.data_ptr(), err=err.data_ptr(),
                                        stream=_stream(torch))
    other = None
    for start in (0, 500, n - M):
        pos.copy_(dev(torch, np.arange(start, start + M, dtype=np.int32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        beside = _prefill(torch, d_q, hq, hkv, dev(torch, np.arange(n - M, n, dtype=np.int32)), slot, d_bt, n_pages,
                          P.E4M3, d_pool, np.array([[0, M]], np.int32), err)
        torch.cuda.synchronize()
        assert other is None or torch.equal(other, beside)
        other = beside
        got = out.cpu().numpy()
        for m in range(0, M, 7):
            k, v = (x[0] for x in P.read(pool, bt[0], 0, start + m + 1, P.E4M3))
            assert rel_rms(got[m], P.attention(q[m], k, v).reshape(-1)) <= 5e-6
    assert torch.equal(out, other) and int(err) == 0


# ---------------------------------------------------------------- together --
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_a_layers_steps_together_and_from_a_graph(torch_cuda, fmt):
    """A prompt chunk through kernel (1) and the prefill attention, then decode steps (one row
    per sequence, one of them padding) from ONE captured graph whose positions advance on the
    device, on a stream of its own; every output against the read-back of the pages."""
    torch = torch_cuda
    rng = np.random.default_rng(11)
    hq, hkv, max_pos, lens = 16, 8, 256, [45, 16, 70]
    n_steps, n_pages = 20, 24
    rope = np.asarray(oracle.rope_table(max_pos), np.float32).reshape(max_pos, 64, 2)
    bt = _table(rng, [n + n_steps for n in lens], n_pages)
    qn, kn = (rng.uniform(0.8, 1.2, 128).astype(np.float32) for _ in range(2))
    pool, err = dev(torch, _garbage_pool(rng, 1, n_pages, hkv)), _err(torch)
    d_bt, d_rope, d_qn, d_kn = (dev(torch, a) for a in (bt, rope, qn, kn))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def kernel1(qkv, pos, slot, q):
        fa_dec.op_qknorm_rope_append_kv8(qkv.data_ptr(), len(pos), hq, hkv, pos.data_ptr(), slot.data_ptr(),
                                         d_bt.data_ptr(), bt.shape[1], n_pages, d_qn.data_ptr(), d_kn.data_ptr(), 1e-5,
                                         d_rope.data_ptr(), max_pos, fmt, pool.data_ptr(), q.data_ptr(),
                                         err.data_ptr(), _stream(torch))

    def check(out, q, pos, slot):
        host = pool.cpu().numpy()
        for m in range(len(pos)):
            if pos[m] < 0:
                assert not out[m].any()
                continue
            k, v = (x[0] for x in P.read(host, bt[slot[m]], 0, pos[m] + 1, fmt))
            assert rel_rms(out[m], P.attention(q[m], k, v).reshape(-1)) <= 5e-6, (m, pos[m])

    with torch.cuda.stream(side):
        pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
        slot = np.repeat([0, 1, 2], lens).astype(np.int32)
        qkv = dev(torch, _vectors(rng, len(pos), hq + 2 * hkv))
        q = torch.zeros((len(pos), hq, 128), device="cuda")
        d_pos, d_slot = dev(torch, pos), dev(torch, slot)
        kernel1(qkv, d_pos, d_slot, q)
        first = np.concatenate([[0], np.cumsum(lens)[:-1]])
        out = _prefill(torch, q, hq, hkv, d_pos, d_slot, d_bt, n_pages, fmt, pool,
                       _tiles([(int(f), n) for f, n in zip(first, lens)], 64), err)
        side.synchronize()
        check(out.cpu().numpy(), q.cpu().numpy(), pos, slot)

        M = 4
        d_pos = dev(torch, np.array(lens + [-1], np.int32))
        d_slot = dev(torch, np.array([0, 1, 2, 0], np.int32))
        step = dev(torch, np.array([1, 1, 1, 0], np.int32))
        qkv = torch.zeros((M, hq + 2 * hkv, 128), device="cuda")
        q, out = torch.zeros((M, hq, 128), device="cuda"), torch.zeros((M, hq * 128), device="cuda")
        size = fa_dec.op_attention_kv8_scratch_bytes(M, hq, hkv)
        scratch = _scratch(torch, size)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kernel1(qkv, d_pos, d_slot, q)
            fa_dec.op_paged_attention_kv8(q.data_ptr(), M, hq, hkv, d_pos.data_ptr(), d_slot.data_ptr(),
                                          d_bt.data_ptr(), bt.shape[1], n_pages, fmt, pool.data_ptr(),
                                          scratch.data_ptr(), size, out32=out.data_ptr(), err=err.data_ptr(),
                                          stream=_stream(torch))
            d_pos += step
        for i in range(n_steps):
            qkv.copy_(dev(torch, _vectors(rng, M, hq + 2 * hkv)))
            graph.replay()
            side.synchronize()
            if i % 6 == 0 or i == n_steps - 1:
                check(out.cpu().numpy(), q.cpu().numpy(), np.array([n + i for n in lens] + [-1]), [0, 1, 2, 0])
    assert int(err) == 0


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_bytes_do_not_depend_on_how_tokens_are_cut_into_calls(torch_cuda, fmt):
    torch = torch_cuda
    rng = np.random.default_rng(12)
    M, hkv = 50, 8
    k, v = dev(torch, _vectors(rng, M, 2, hkv)), dev(torch, _vectors(rng, M, 2, hkv))
    pos, slot = dev(torch, np.arange(M, dtype=np.int32)), dev(torch, np.zeros(M, np.int32))
    bt = dev(torch, np.array([[3, 0, 2, 1]], np.int32))
    pools = []
    for cuts in ([0, 50], [0, 1, 2, 17, 18, 40, 50]):
        pool, err = torch.zeros((2, 4, hkv, P.TILE), dtype=torch.uint8, device="cuda"), _err(torch)
        for a, b in zip(cuts, cuts[1:]):
            _append(torch, k[a:b], v[a:b], P.F32, 2 * hkv * 128, b - a, 2, hkv, pos[a:b].contiguous(), slot, bt, 4,
                    fmt, pool, err)
        pools.append(pool)
        assert int(err) == 0
    assert torch.equal(*pools)


def test_two_decode_calls_on_two_streams(torch_cuda):
    """Calls with scratch of their own may overlap; results repeat bit for bit."""
    torch = torch_cuda
    rng = np.random.default_rng(13)
    hq, hkv, lens = 16, 8, [900, 1200, 3]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, P.INT8)
    d_pool, d_bt = dev(torch, pool), dev(torch, bt)
    pos, slot = dev(torch, np.array(lens, np.int32) - 1), dev(torch, np.arange(3, dtype=np.int32))
    qs = [dev(torch, (rng.standard_normal((3, hq, 128)) * 0.3).astype(np.float32)) for _ in range(2)]
    err = _err(torch)
    alone = [_decode(torch, q, hq, hkv, pos, slot, d_bt, n_pages, P.INT8, d_pool, err) for q in qs]
    outs = [torch.zeros((3, hq * 128), device="cuda") for _ in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    keep = []
    for _ in range(20):
        for s, q, o in zip(streams, qs, outs):
            with torch.cuda.stream(s):
                keep.append(_decode(torch, q, hq, hkv, pos, slot, d_bt, n_pages, P.INT8, d_pool, err, out=o))
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert torch.equal(a, b)
    assert int(err) == 0


# ------------------------------------------------------------ large scores --
def _one_hot_rows(got, q, pos, pool, bt, fmt):
    """Checks got [M][Hq][128] of rows whose scores are far larger than 1 (sequence 0): every
    output is finite and within the values that its row attends to, and where the definition
    gives the largest score all the weight, the output is that token's value. A score is off by
    2^-18 of sum |q k| at most (see _bound), two of them by twice that; a lead of 40 beyond it
    leaves the others e^-40 each. An output is then the weight's pair (2^-22), the division and
    a few f32 roundings away from the value, and a pair's smallest step from that of the largest
    V: 2^-20 of it together. Returns the share of (row, head)s with such a lead."""
    M, hq, clear = len(q), q.shape[1], 0
    for m in range(M):
        k, v = (x[0] for x in P.read(pool, bt[0], 0, pos[m] + 1, fmt))
        g = hq // len(k)
        for h in range(hq):
            kh, vh, qh = k[h // g], v[h // g], q[m, h].astype(np.float64)
            tol = 2.0 ** -20 * np.abs(vh).max()
            assert np.isfinite(got[m, h]).all(), (m, h)
            assert (got[m, h] <= vh.max(0) + tol).all() and (got[m, h] >= vh.min(0) - tol).all(), (m, h)
            s = kh @ qh
            lead = np.sort(s)[-1] - np.sort(s)[-2] if len(s) > 1 else np.inf
            if lead >= 2.0 ** -17 * (np.abs(kh) @ np.abs(qh)).max() + 40:
                clear += 1
                assert np.abs(got[m, h] - vh[s.argmax()]).max() <= tol, (m, h)
    return clear / (M * hq)


@pytest.mark.parametrize("size", [1e4, 1e6, 1e7, 1e8, 3e8, 1e9, 1e10, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_large_scores(torch_cuda, fmt, which, size):
    """Scores of 1e4 to 1e31: the maximum that a kernel takes off them is theirs, not a rounded one."""
    torch = torch_cuda
    rng = np.random.default_rng(31)
    hq, hkv, n, M = 16, 8, 300, 20
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    q = (rng.standard_normal((M, hq, 128)) * 0.3 * size).astype(np.float32)
    pos = np.arange(n - M, n).astype(np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = _decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)
    assert int(err) == 0
    assert _one_hot_rows(got.cpu().numpy().reshape(M, hq, 128), q, pos, pool, bt, fmt) > 0.9


@pytest.mark.parametrize("base,M", [(0, 70), (37, 64), (1000, 20)])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_rows_that_see_large_keys_and_values(torch_cuda, fmt, which, base, M):
    """K and V of 1e30 in the second half of a chunk, for the rows that attend to them."""
    torch = torch_cuda
    rng = np.random.default_rng(base + M)
    hq, hkv, n = 16, 8, base + M
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    _, scales = P.parts(pool)
    late = np.arange(base + M // 2, n)
    for part in (0, 1):
        scales[0, bt[0, late // 16], :, part, late % 16] *= np.float32(1e30)
    pos = np.arange(base, n).astype(np.int32)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = _decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)
    assert int(err) == 0
    at = np.arange(M // 2, M)
    assert _one_hot_rows(got.cpu().numpy().reshape(M, hq, 128)[at], q[at], pos[at], pool, bt, fmt) > 0.8      # the first rows see few such keys


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_scores_past_f32_are_nan(torch_cuda, fmt, which):
    """A row whose largest score passes f32's range has no finite answer, least of all zeros."""
    torch = torch_cuda
    rng = np.random.default_rng(32)
    hq, hkv, n, M = 16, 8, 130, 4
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    _, scales = P.parts(pool)
    t = np.arange(n)
    scales[0, bt[0, t // 16], :, 0, t % 16] *= np.float32(1e25)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    q[:, ::2] *= np.float32(1e25)                                 # the even heads: scores of 1e50; the odd ones 1e25
    pos = np.full(M, n - 1, np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = (_decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)).cpu().numpy()
    got = got.reshape(M, hq, 128)
    assert np.isnan(got[:, ::2]).all() and np.isfinite(got[:, 1::2]).all() and int(err) == 0


@pytest.mark.parametrize("period", [16, 64, 128])
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_large_scores_that_rise_by_their_last_place(torch_cuda, fmt, which, period):
    """Scores of 1e8, whose last place is 16 in log2 units, rising by it: a step is more than a
    kernel may leave its running maximum behind, though the sum of the two may round to it."""
    torch = torch_cuda
    rng = np.random.default_rng(33)
    hq, hkv, n, M = 16, 8, 1024, 20
    pool, bt, n_pages = _filled(rng, [n], 1, hkv, fmt)
    raw, scales = P.parts(pool)
    t = np.arange(n)
    # K: the largest stored value in dimension 0 alone, under scales that rise by one step of f32
    top = 127.0 if fmt == P.INT8 else 448.0
    raw[0, bt[0, t // 16], :, 0, t % 16] = 0
    raw[0, bt[0, t // 16], :, 0, t % 16, 0] = 127 if fmt == P.INT8 else 126
    d = (np.float32(1.03).view(np.int32) + (t + 40) // period).astype(np.int32).view(np.float32)
    scales[0, bt[0, t // 16], :, 0, t % 16] = d[:, None]
    q = np.zeros((M, hq, 128), np.float32)
    q[..., 0] = np.linspace(0.94e8, 1.85e8, M * hq).reshape(M, hq) / (top * 1.03)      # in log2 units 2^27 to 2^28
    pos = np.full(M, n - 1, np.int32)
    args = (torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, np.zeros(M, np.int32)), dev(torch, bt), n_pages,
            fmt, dev(torch, pool))
    err = _err(torch)
    got = _decode(*args, err) if which == "decode" else _prefill(*args, _tiles([(0, M)], 64), err)
    assert int(err) == 0
    _one_hot_rows(got.cpu().numpy().reshape(M, hq, 128), q, pos, pool, bt, fmt)


# -------------------------------------------------- keys of any magnitude --
@pytest.mark.parametrize("eps,size", [(1e-5, 1.0), (0.0, 1.0), (1e-5, 1e-37), (1e-5, 3e37), (1e-5, 3e38)])
@pytest.mark.parametrize("M", [100, 600])                         # a key vector a warp, and several
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_qknorm_rope_append_keys_of_any_magnitude(torch_cuda, fmt, M, eps, size):
    """K's bytes are those of 64 bits where f32 squares overflow or vanish, where the norm weights
    take the values next to f32's limits, and for zero, infinite and NaN vectors."""
    torch = torch_cuda
    rng = np.random.default_rng(M)
    hq, hkv, max_pos, eps = 1, 8, 640, np.float32(eps)
    qkv = _vectors(rng, M, hq + 2 * hkv)
    mag = 10.0 ** rng.uniform(-42, 36, (M, hkv, 1))
    qkv[:, hq:hq + hkv] = (qkv[:, hq:hq + hkv] * mag).astype(np.float32)
    qkv[1, hq], qkv[2, hq + 1, 5], qkv[3, hq + 2, 100], qkv[4, hq + 3, 0] = 0, np.inf, np.nan, -np.inf
    qkv[5, hq + 4] = np.finfo(np.float32).max
    kn = (rng.uniform(0.8, 1.1, 128) * size).astype(np.float32)
    assert np.isfinite(kn).all()
    rope = np.asarray(oracle.rope_table(max_pos), np.float32).reshape(max_pos, 64, 2)
    pos, n_pages = np.arange(M, dtype=np.int32), max_pos // 16
    bt = rng.permutation(n_pages).astype(np.int32)[None]
    pool, err = torch.zeros((1, n_pages, hkv, P.TILE), dtype=torch.uint8, device="cuda"), _err(torch)
    q = torch.zeros((M, hq, 128), device="cuda")
    d = [dev(torch, a) for a in (qkv, pos, np.zeros(M, np.int32), bt, np.ones(128, np.float32), kn, rope)]
    p = [x.data_ptr() for x in d]
    fa_dec.op_qknorm_rope_append_kv8(p[0], M, hq, hkv, p[1], p[2], p[3], n_pages, n_pages, p[4], p[5], float(eps),
                                     p[6], max_pos, fmt, pool.data_ptr(), q.data_ptr(), err.data_ptr(),
                                     _stream(torch))
    with np.errstate(all="ignore"):
        y = P.norm_rotate_exact(qkv[:, hq:hq + hkv], kn, rope[:M], eps)
    y = np.where(np.abs(y) > np.finfo(np.float32).max, np.inf, y)
    want, d_want = P.quantise(np.where(np.isnan(y), np.inf, y), fmt)
    raw, scales = P.parts(pool.cpu().numpy())
    at = bt[0, pos // 16], pos % 16
    got, d_got = raw[0, at[0], :, 0, at[1]], scales[0, at[0], :, 0, at[1]]
    assert np.array_equal(np.isnan(d_got), np.isnan(d_want)) and np.isnan(d_want).any() and not np.isnan(d_want).all()
    assert np.array_equal(got, want)
    live = ~np.isnan(d_want)
    off = np.abs(d_got[live].astype(np.float64) - d_want[live])
    assert (off <= d_want[live].astype(np.float64) * (2.0 ** -20 if fmt == P.INT8 else 0)).all()
    v, d_v = P.quantise(qkv[:, hq + hkv:], fmt)
    assert np.array_equal(raw[0, at[0], :, 1, at[1]], v) and np.array_equal(scales[0, at[0], :, 1, at[1]], d_v)
    assert int(err) == 0


# -------------------------------------------------- forms of the large calls --
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("src_type,layers,hkv,M", [(P.F16, 4, 8, 300), (P.F32, 3, 11, 300), (P.BF16, 1, 5, 2000),
                                                   (P.F32, 28, 8, 45), (P.BF16, 2, 8, 601), (P.F16, 1, 1, 9500)])
def test_append_of_many_vectors(torch_cuda, fmt, src_type, layers, hkv, M):
    """Calls in which a warp takes several (layer, head) pairs: rows whose pairs do not fill a warp,
    padding, a bad position and a bad page among them; bytes and error bits in full."""
    torch = torch_cuda
    rng = np.random.default_rng(M)
    n_pages = -(-M // 16) + 2
    bt = rng.permutation(n_pages)[:-(-M // 16)].astype(np.int32)[None]
    pos, kb = rng.permutation(M).astype(np.int32), bt.copy()
    want = pos.copy()
    pos[[1, M // 2]] = want[[1, M // 2]] = -1
    pos[M - 1], want[M - 1] = -7, -1
    kb[0, 1] = n_pages
    want[(want >= 16) & (want < 32)] = -1
    ld, n = 2 * layers * hkv * 128 + 64, layers * hkv * 128
    x = np.zeros((M, ld), np.float32)
    x[:, :n], x[:, n:2 * n] = _vectors(rng, M, layers * hkv).reshape(M, n), _vectors(rng, M, layers * hkv).reshape(M, n)
    x[0, :128], x[M // 3, n + 5] = 0, 1000
    d_x, x = _src(torch, x, src_type)
    k, v = (x[:, i * n:(i + 1) * n].reshape(M, layers, hkv, 128) for i in (0, 1))
    pool, slot = _garbage_pool(rng, layers, n_pages, hkv), np.zeros(M, np.int32)
    d_pool, d_err = dev(torch, pool), _err(torch)
    _append(torch, d_x, d_x[:, n:], src_type, ld, M, layers, hkv, dev(torch, pos), dev(torch, slot), dev(torch, kb),
            n_pages, fmt, d_pool, d_err)
    P.write(pool, bt, slot, want, k, v, fmt)
    assert np.array_equal(d_pool.cpu().numpy(), pool)
    assert int(d_err) == 2 | 4


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,M", [(16, 8, 400), (12, 4, 500), (5, 5, 700), (16, 2, 480), (1, 1, 3200), (3, 1, 1999)])
def test_qknorm_rope_append_of_many_rows(torch_cuda, fmt, hq, hkv, M):
    """Calls in which a warp takes several head vectors: warps of queries, of keys, of values and
    mixed ones; q_out, bytes, scales, padding and error bits in full."""
    torch = torch_cuda
    rng = np.random.default_rng(hq * 100 + M)
    max_pos = -(-M // 16) * 16 + 16
    n_pages = max_pos // 16 + 3
    qkv = _vectors(rng, M, hq + 2 * hkv) * 2
    qkv[0, hq] = 0
    qn, kn = (rng.uniform(0.8, 1.2, 128).astype(np.float32) for _ in range(2))
    rope = np.asarray(oracle.rope_table(max_pos), np.float32).reshape(max_pos, 64, 2)
    bt = _table(rng, [max_pos], n_pages)
    pos = rng.permutation(max_pos)[:M].astype(np.int32)
    slot = np.zeros(M, np.int32)
    pos[1], slot[1] = -1, 10 ** 6                                 # padding
    pos[2], pos[3] = -9, max_pos                                  # bad
    slot[4] = -1                                                  # bad: appends nothing
    pool = _garbage_pool(rng, 1, n_pages, hkv)
    d_pool, d_err = dev(torch, pool), _err(torch)
    q_out = torch.full((M, hq, 128), 7.0, device="cuda")
    d = [dev(torch, a) for a in (qkv, pos, slot, bt, qn, kn, rope)]
    p = [x.data_ptr() for x in d]
    fa_dec.op_qknorm_rope_append_kv8(p[0], M, hq, hkv, p[1], p[2], p[3], bt.shape[1], n_pages, p[4], p[5], 1e-5, p[6],
                                     max_pos, fmt, d_pool.data_ptr(), q_out.data_ptr(), d_err.data_ptr(),
                                     _stream(torch))
    rot = rope[np.clip(pos, 0, max_pos - 1)]
    q = P.norm_rotate(qkv[:, :hq], qn, rot) * np.float32(1 / np.sqrt(np.float32(128)))
    q[1:4] = 7
    got_q, rest = q_out.cpu().numpy(), np.r_[0:4, 5:M]
    assert np.array_equal(got_q[rest], q[rest])
    want = np.where(slot < 0, -1, np.where(pos < max_pos, pos, -1))
    k = P.norm_rotate_exact(qkv[:, hq:hq + hkv], kn, rot)
    P.write(pool, bt, np.zeros(M, np.int32), want, k[:, None], qkv[:, hq + hkv:][:, None], fmt)
    (raw, d), (raw_w, d_w) = P.parts(d_pool.cpu().numpy()), P.parts(pool)
    assert np.array_equal(raw, raw_w)
    assert np.array_equal(d[..., 1, :].view(np.uint32), d_w[..., 1, :].view(np.uint32))
    live = np.isfinite(d_w[..., 0, :])
    assert np.array_equal(live, np.isfinite(d[..., 0, :]))
    off = np.abs(d[..., 0, :][live].astype(np.float64) - d_w[..., 0, :][live])
    assert (off <= np.abs(d_w[..., 0, :][live]) * (2.0 ** -20 if fmt == P.INT8 else 0)).all()
    assert int(d_err) == 4


@pytest.mark.parametrize("step", [0.0, 0.002, -0.002, 0.05, -0.05])
@pytest.mark.parametrize("blocks", [(33, 70), (64, 65)])
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_prefill_attention_many_tiles_over_long_contexts(torch_cuda, fmt, blocks, step):
    """Calls of enough tiles that no context is cut into parts, over more than 32 blocks of 64 keys
    (whose products are joined 32 blocks at a time, the last time one, six or 32 of them), with
    scores that stay, rise or fall along the context."""
    torch = torch_cuda
    rng = np.random.default_rng(blocks[0])
    hq, hkv, per = 16, 8, 3
    lens = [64 * b for b in blocks]
    pool, bt, n_pages = _filled(rng, lens, 1, hkv, fmt)
    q = rng.standard_normal((10 * per, hq, 128)) * 0.3
    if step:
        raw, scales = P.parts(pool)
        way = rng.choice([-1.0, 1.0], 128)
        q = way + 0.01 * q
        for i, n in enumerate(lens):
            t = np.arange(n)
            k = way * (step * t / 128)[:, None] + 0.02 * rng.standard_normal((hkv, n, 128))
            qk, dk = P.quantise(k.astype(np.float32), fmt)
            raw[0, bt[i, t // 16], :, 0, t % 16] = qk.transpose(1, 0, 2)
            scales[0, bt[i, t // 16], :, 0, t % 16] = dk.T
    q = q.astype(np.float32)
    slot = np.repeat(np.arange(10) % 2, per).astype(np.int32)     # ten tiles of three rows
    pos = np.array([lens[s] - per + m % per for m, s in enumerate(slot)], np.int32)
    tiles = _tiles([(per * i, per) for i in range(10)], 64)
    assert fa_dec.op_prefill_attention_kv8_scratch_bytes(len(tiles), hq, hkv) == 0
    err = _err(torch)
    got = _prefill(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
                   dev(torch, pool), tiles, err).cpu().numpy()
    assert int(err) == 0
    for m in range(len(pos)):
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, fmt))
        want = P.attention(q[m], k, v).reshape(-1)
        assert np.abs(got[m] - want).max() <= _bound(q[m], k, v), m
        if abs(step) < 0.05:
            assert rel_rms(got[m], want) <= 5e-6, m


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,M,pages", [
    (16, 8, 1, 32), (16, 8, 9, 64), (16, 8, 9, 65), (16, 8, 18, 64), (16, 8, 19, 20), (16, 8, 55, 9), (16, 8, 56, 9),
    (32, 4, 30, 12), (32, 4, 50, 12), (7, 1, 100, 3), (16, 8, 700, 8), (64, 64, 9, 57), (8, 2, 1500, 4),
    (200, 200, 3, 10)])
def test_decode_attention_counts_every_token(torch_cuda, fmt, hq, hkv, M, pages):
    """Each way of cutting a call into work, at an accuracy that a token lost or taken twice
    exceeds: one of 1024 tokens moves a row by some 1e-3 of itself."""
    torch = torch_cuda
    rng = np.random.default_rng(100 * pages + M)
    lens = rng.integers(1, 16 * pages + 1, min(M, 24))
    lens[0] = 16 * pages
    pool, bt, n_pages = _filled(rng, lens.tolist(), 1, hkv, fmt)
    slot = (np.arange(M) % len(lens)).astype(np.int32)
    pos = (lens[slot] - 1).astype(np.int32)
    q = (rng.standard_normal((M, hq, 128)) * 0.3).astype(np.float32)
    err = _err(torch)
    got = _decode(torch, dev(torch, q), hq, hkv, dev(torch, pos), dev(torch, slot), dev(torch, bt), n_pages, fmt,
                  dev(torch, pool), err).cpu().numpy()
    assert int(err) == 0
    for m in np.unique(np.r_[np.arange(0, M, max(1, M // 24)), M - 1]):
        k, v = (x[0] for x in P.read(pool, bt[slot[m]], 0, pos[m] + 1, fmt))
        assert rel_rms(got[m], P.attention(q[m], k, v).reshape(-1)) <= 5e-6, (m, pos[m])
