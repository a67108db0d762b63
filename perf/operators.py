"""Workloads of the 8-bit paged KV cache: writing it, reading it back, and attention over it.

One page of one layer holds 16 tokens of a sequence: for each KV head 4224 bytes, K [16][128]
and V [16][128] in 8 bits (int8 or e4m3), then the f32 scales of the 16 K and of the 16 V
vectors. A vector x is stored with a scale d and the values x / d:
  int8  d = max(amax / 127, 2^-126) in f32, x / d rounded to the nearest integer, ties to even
  e4m3  d = the smallest power of two >= 2^-126 with amax <= 448 d, x / d rounded to e4m3
`listed()` gives the standing cases, `draw()` more of the same ranges; `run()` makes one pass
with the library's entry points (own) or in plain torch operations.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

D = 128            # head dimension
PAGE = 16          # tokens per page
TILE = 4224        # bytes of one KV head in one page
INT8, E4M3 = 0, 1
TINY = 2.0 ** -126
EPS = 1e-5
ROPE_BASE = 1e6
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
FORMATS = {"int8": INT8, "e4m3": E4M3}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one stream's decode step: its token's K/V in all 28 layers, written and read back
        dict(name="append 1 token", op="append", format="int8", type="f16", heads=16, kv_heads=8, layers=28, seqs=1,
             shortest=1, longest=1, before=255),
        # 16 prompts of mixed lengths written at once (8 layers), from f32 activations
        dict(name="append 16 prompts", op="append", format="e4m3", type="f32", heads=16, kv_heads=8, layers=8,
             seqs=16, shortest=37, longest=517, before=5),
        # the decode step's form of one layer: one row through norm, rotation and the cache
        dict(name="norm append 1 row", op="norm_append", format="int8", type="f16", heads=16, kv_heads=8, layers=1,
             seqs=1, shortest=1, longest=1, before=112),
        # the largest forward of the decoder (4096 rows): eight prompts of 512 rows
        dict(name="norm append 4096 rows", op="norm_append", format="e4m3", type="f16", heads=16, kv_heads=8,
             layers=1, seqs=8, shortest=512, longest=512, before=0),
        # 32 short streams read back over all layers into the contiguous cache view
        dict(name="read back 32 streams", op="read_back", format="int8", type="f16", heads=16, kv_heads=8, layers=28,
             seqs=32, shortest=1, longest=320, before=0),
        # one long stream read back, bf16
        dict(name="read back 4001 tokens", op="read_back", format="e4m3", type="bf16", heads=16, kv_heads=8,
             layers=28, seqs=1, shortest=4001, longest=4001, before=7),
        # one stream early in its decode: latency
        dict(name="decode 1 x 256", op="decode", format="int8", type="f32", heads=16, kv_heads=8, layers=1, seqs=1,
             shortest=256, longest=256, before=0),
        # a small batch of streams at different places, odd lengths
        dict(name="decode 16 x 1..1021", op="decode", format="e4m3", type="f32", heads=16, kv_heads=8, layers=1,
             seqs=16, shortest=1, longest=1021, before=0),
        # the serving batch: 128 streams at 2048 tokens
        dict(name="decode 128 x 2048", op="decode", format="int8", type="f32", heads=16, kv_heads=8, layers=1,
             seqs=128, shortest=2048, longest=2048, before=0),
        # one stream at the longest context, eight query heads to a KV head
        dict(name="decode 1 x 40960", op="decode", format="int8", type="f16", heads=32, kv_heads=4, layers=1, seqs=1,
             shortest=40960, longest=40960, before=0),
        # one utterance's prompt of 112 rows
        dict(name="prefill 112 rows", op="prefill", format="int8", type="f32", heads=16, kv_heads=8, layers=1, seqs=1,
             shortest=112, longest=112, before=0),
        # chunks of four prompts over what they have cached already
        dict(name="prefill 4 x 512 at 3500", op="prefill", format="e4m3", type="f32", heads=16, kv_heads=8, layers=1,
             seqs=4, shortest=417, longest=512, before=3500),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "norm_append", "read_back", "decode", "decode", "prefill"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (16, 8), (8, 8), (12, 4), (16, 2), (32, 8), (5, 5)])
    case = dict(op=op, format=rng.choice(["int8", "e4m3"]), type="f32", heads=heads, kv_heads=kv_heads, layers=1)
    if op in ("append", "read_back"):
        case.update(type=rng.choice(["f16", "bf16", "f32"]), layers=_log_int(rng, 1, 28))
        budget = 100000 // (case["layers"] * kv_heads // 2 + 1)
    elif op == "norm_append":
        case.update(type=rng.choice(["f16", "bf16"]))
        budget = 4096
    elif op == "decode":
        budget = 128 * 2048 * 4 // max(4, kv_heads)
    else:
        budget = 1500
    case["seqs"] = _log_int(rng, 1, 128 if op == "decode" else 32 if op != "prefill" else 6)
    case["longest"] = _log_int(rng, 1, max(1, min(40960 if op == "decode" else 2048, budget // case["seqs"])))
    case["shortest"] = _log_int(rng, 1, case["longest"])
    case["before"] = 0 if op == "decode" or rng.random() < 0.3 else _log_int(rng, 1, 3000)
    return case


def _lengths(case):
    """Tokens of each sequence, spread between the shortest and the longest; the first is the longest."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    return [hi - ((hi - lo) * ((7 * i) % n)) // max(1, n - 1) for i in range(n)]


def work(case):
    lens, layers, hq, hkv, before = _lengths(case), case["layers"], case["heads"], case["kv_heads"], case["before"]
    size = torch.empty(0, dtype=TYPES[case["type"]][1]).element_size()
    n = sum(lens)
    vectors = n * layers * hkv * 2
    stored = vectors * (D + 4)
    if case["op"] == "append":      # the source once, the cache once out and once in, the values read back
        return dict(bytes=vectors * D * (size + 2) + 2 * stored, flops=vectors * D * 4)
    if case["op"] == "norm_append":
        rows = n * (2 * hq + 2 * hkv) * D * 4 + n * D * 4
        return dict(bytes=rows + vectors * D * size + 2 * stored, flops=n * (hq + 2 * hkv) * D * 8)
    if case["op"] == "read_back":
        return dict(bytes=stored + vectors * D * size, flops=vectors * D)
    if case["op"] == "decode":
        return dict(bytes=stored + case["seqs"] * hq * D * 8, flops=4 * n * hq * D)
    keys = sum(m * before + m * (m + 1) // 2 for m in lens)
    cached = sum(m + before for m in lens) * hkv * 2 * (D + 4)
    return dict(bytes=cached + n * hq * D * 8, flops=4 * keys * hq * D)


# ----------------------------------------------------------------- inputs --
def _i32(values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def _scale(amax, fmt):
    """The f32 scale of vectors with these largest magnitudes."""
    if fmt == INT8:
        return (amax.double() / 127).float().clamp_min(TINY)
    m, e = torch.frexp(amax.float())
    k = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126)
    return torch.ldexp(torch.ones_like(m), torch.where(amax > 0, k, torch.full_like(k, -126)))


def _quantise(x, fmt):
    """Stored bytes and scales of x [..., 128]; the quotients in 64 bits, so that none crosses a border."""
    x = x.double()
    d = _scale(x.abs().amax(-1), fmt)
    y = x / d.double()[..., None]
    if fmt == INT8:
        return torch.round(y).to(torch.int8).view(torch.uint8), d
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8), d   # x / d is exact in 32 bits: d is a power of two


def _values(raw, fmt, dtype=torch.float32):
    return raw.view(torch.int8 if fmt == INT8 else torch.float8_e4m3fn).to(dtype)


def _parts(pool):
    """Views of a pool [layers][pages][kv heads][4224]: bytes [..., K|V, token, 128] and scales [..., K|V, token]."""
    raw = pool[..., : 2 * PAGE * D].unflatten(-1, (2, PAGE, D))
    scales = pool[..., 2 * PAGE * D:].view(torch.float32).unflatten(-1, (2, PAGE))
    return raw, scales


def _rope(n):
    inv = ROPE_BASE ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device="cuda") / D)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    op, fmt, hq, hkv, layers = case["op"], FORMATS[case["format"]], case["heads"], case["kv_heads"], case["layers"]
    lens, before, n_seq = _lengths(case), case["before"], case["seqs"]
    total = [m + before for m in lens]
    stride = -(-max(total) // PAGE)
    n_pages = sum(-(-t // PAGE) for t in total) + 3
    order = host.permutation(n_pages)
    table, used = np.zeros((n_seq, stride), np.int32), 0
    for i, t in enumerate(total):
        need = -(-t // PAGE)
        table[i, :need] = order[used:used + need]
        used += need
    n = sum(lens)
    code, dtype = TYPES[case["type"]]
    s = dict(op=op, fmt=fmt, hq=hq, hkv=hkv, layers=layers, n=n, n_seq=n_seq, lens=lens, before=before, stride=stride,
             n_pages=n_pages, longest=case["longest"], code=code, dtype=dtype, table=torch.tensor(table, device="cuda"),
             err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    first = np.concatenate([[0], np.cumsum(lens)[:-1]])
    slot = np.repeat(np.arange(n_seq), lens)
    pos = np.concatenate([before + np.arange(m) for m in lens])
    s["slot"], s["pos"] = _i32(slot), _i32(pos)
    s["seq"], s["t0"], s["count"], s["row0"] = (_i32(np.arange(n_seq)), _i32([before] * n_seq), _i32(lens), _i32(first))

    def activations(*shape):   # vectors of different sizes with a few large channels, as keys and values have them
        x = torch.randn(*shape, D, generator=g, device="cuda")
        x *= torch.exp(0.4 * torch.randn(*shape, 1, generator=g, device="cuda"))
        x[..., ::37] *= 4
        return x

    s["pool"] = torch.randint(0, 256, (layers, n_pages, hkv, TILE), generator=g, dtype=torch.uint8, device="cuda")
    raw, scales = _parts(s["pool"])
    if op in ("append", "norm_append"):
        scales.fill_(1.0)
    else:   # a filled cache, layer by layer
        for layer in range(layers):
            for page in range(0, n_pages, 4096):
                part = raw[layer, page:page + 4096]
                q, d = _quantise(activations(*part.shape[:-1]).half(), fmt)
                part.copy_(q)
                scales[layer, page:page + 4096] = d
    if op == "append":
        s["k"], s["v"] = (activations(n, layers, hkv).to(dtype).contiguous() for _ in range(2))
    if op == "norm_append":
        s["qkv"] = 2 * activations(n, hq + 2 * hkv)
        s["qn"], s["kn"] = (0.8 + 0.4 * torch.rand(D, generator=g, device="cuda") for _ in range(2))
        s["rope"] = _rope(max(total))
        s["q_out"] = torch.empty(n, hq, D, device="cuda")
    if op in ("append", "norm_append", "read_back"):
        out = dtype if op != "append" else torch.float16
        s["out_code"] = code if op != "append" else TYPES["f16"][0]
        s["k_out"], s["v_out"] = (torch.zeros(layers, hkv, n, D, dtype=out, device="cuda") for _ in range(2))
    if op == "decode":
        s["rows"], s["row_slot"], s["row_pos"] = n_seq, s["seq"], _i32([m - 1 for m in lens])
    if op == "prefill":
        s["rows"], s["row_slot"], s["row_pos"] = n, s["slot"], s["pos"]
        step = 128 * hkv // hq
        tiles = [(f + i, min(step, m - i)) for f, m in zip(first, lens) for i in range(0, m, step)]
        s["tiles"], s["n_tiles"] = _i32(tiles), len(tiles)
        s["place"] = _i32(np.arange(n) - first[slot])
    if op in ("decode", "prefill"):
        s["q"] = activations(s["rows"], hq) * (0.9 / math.sqrt(D))
        s["out"] = torch.zeros(s["rows"], hq * D, dtype=dtype, device="cuda")
    return s


# -------------------------------------------------------- the library's calls --
def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "funasr-ggml_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fa_dec
    return fa_dec


def _run_own(s):
    fa = _library()
    stream = torch.cuda.current_stream().cuda_stream
    fmt, hq, hkv, table, err = s["fmt"], s["hq"], s["hkv"], s["table"].data_ptr(), s["err"].data_ptr()
    pool, slot, pos = s["pool"].data_ptr(), s["slot"].data_ptr(), s["pos"].data_ptr()
    if s["op"] == "append":
        fa.op_kv8_append(s["k"].data_ptr(), s["v"].data_ptr(), s["code"], s["layers"] * hkv * D, s["n"], s["layers"],
                         hkv, pos, slot, table, s["stride"], s["n_pages"], fmt, pool, err, stream)
    if s["op"] == "norm_append":
        fa.op_qknorm_rope_append_kv8(s["qkv"].data_ptr(), s["n"], hq, hkv, pos, slot, table, s["stride"], s["n_pages"],
                                     s["qn"].data_ptr(), s["kn"].data_ptr(), EPS, s["rope"].data_ptr(),
                                     s["rope"].shape[0], fmt, pool, s["q_out"].data_ptr(), err, stream)
    if s["op"] in ("append", "norm_append", "read_back"):
        fa.op_kv8_gather(pool, fmt, s["layers"], s["n_pages"], hkv, table, s["stride"], s["seq"].data_ptr(),
                         s["t0"].data_ptr(), s["count"].data_ptr(), s["row0"].data_ptr(), s["n_seq"], s["longest"],
                         s["n"], s["out_code"], s["k_out"].data_ptr(), s["v_out"].data_ptr(), err, stream)
        return [s["k_out"], s["v_out"]] + ([s["q_out"]] if s["op"] == "norm_append" else [])
    out = s["out"].data_ptr()
    out32, out16 = (out, 0) if s["dtype"] == torch.float32 else (0, out)
    if "scratch" not in s:   # the workspace that an engine allocates with its other buffers
        size = (fa.op_attention_kv8_scratch_bytes(s["rows"], hq, hkv) if s["op"] == "decode" else
                fa.op_prefill_attention_kv8_scratch_bytes(s["n_tiles"], hq, hkv))
        s["scratch"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    if s["op"] == "decode":
        fa.op_paged_attention_kv8(s["q"].data_ptr(), s["rows"], hq, hkv, s["row_pos"].data_ptr(),
                                  s["row_slot"].data_ptr(), table, s["stride"], s["n_pages"], fmt, pool,
                                  s["scratch"].data_ptr(), s["scratch"].numel(), out16=out16, out32=out32, err=err,
                                  stream=stream)
    else:
        fa.op_prefill_attention_kv8(s["q"].data_ptr(), s["rows"], hq, hkv, s["row_pos"].data_ptr(),
                                    s["row_slot"].data_ptr(), table, s["stride"], s["n_pages"], fmt, pool,
                                    s["tiles"].data_ptr(), s["n_tiles"], s["scratch"].data_ptr(),
                                    s["scratch"].numel(), out16=out16, out32=out32, err=err, stream=stream)
    return [s["out"]]


# ------------------------------------------------------------ plain form --
def _token_places(s):
    """Page and place in the page of every row's token."""
    page = s["table"][s["slot"].long(), (s["pos"] // PAGE).long()].long()
    return page, (s["pos"] % PAGE).long()


def _norm_rotate(x, w, rope):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = y[..., : D // 2], y[..., D // 2:]
    c, sn = rope[:, None, :, 0], rope[:, None, :, 1]
    return torch.cat([a * c - b * sn, a * sn + b * c], -1)


def _write(s, k, v):
    """k, v [tokens][layers][kv heads][128] into the pages."""
    raw, scales = _parts(s["pool"])
    page, t = _token_places(s)
    q, d = _quantise(torch.stack([k, v], 3), s["fmt"])          # [tokens][layers][heads][2]
    raw[:, page, :, :, t] = q
    scales[:, page, :, :, t] = d


def _read(s, dtype):
    raw, scales = _parts(s["pool"])
    page, t = _token_places(s)
    x = _values(raw[:, page, :, :, t], s["fmt"]) * scales[:, page, :, :, t][..., None]   # [tokens][layers][heads][2][128]
    return [x[:, :, :, i].permute(1, 2, 0, 3).to(dtype).contiguous() for i in (0, 1)]


def _attend(s):
    n_seq, hq, hkv, rows = s["n_seq"], s["hq"], s["hkv"], s["rows"]
    raw, scales = _parts(s["pool"][0])
    pages = s["table"].long()
    kv = _values(raw[pages], s["fmt"]) * scales[pages][..., None]          # [seq][page][head][2][16][128]
    kv = kv.permute(3, 0, 2, 1, 4, 5).reshape(2, n_seq, hkv, -1, D)
    per = 1 if s["op"] == "decode" else s["longest"]                       # rows of a sequence, padded
    slot = s["row_slot"].long()
    place = slot.new_zeros(rows) if s["op"] == "decode" else s["place"].long()
    q = s["q"].new_zeros(n_seq, per, hq, D)
    q[slot, place] = s["q"]
    last = torch.full((n_seq, per), -1, dtype=torch.int32, device="cuda")
    last[slot, place] = s["row_pos"]
    q = q.reshape(n_seq, per, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(n_seq, hkv, -1, D)
    score = (q @ kv[0].transpose(-1, -2)).reshape(n_seq, hkv, hq // hkv, per, -1)
    key = torch.arange(score.shape[-1], device="cuda")
    seen = (key <= last[..., None])[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, -torch.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - top), torch.zeros_like(score))
    # a masked token's value takes no part, whatever the page holds behind the last token
    value = torch.where((key <= last.amax(1, keepdim=True))[:, None, :, None], kv[1], torch.zeros_like(kv[1]))
    o = (p.reshape(n_seq, hkv, -1, p.shape[-1]) @ value).reshape(n_seq, hkv, hq // hkv, per, D)
    o = (o / p.sum(-1, keepdim=True)).permute(0, 3, 1, 2, 4).reshape(n_seq, per, hq * D)
    return [o[slot, place].to(s["dtype"])]


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "append":
        _write(s, s["k"], s["v"])
        return _read(s, torch.float16)
    if s["op"] == "norm_append":
        hq, hkv, rope = s["hq"], s["hkv"], s["rope"][s["pos"].long()]
        q = _norm_rotate(s["qkv"][:, :hq], s["qn"], rope) / math.sqrt(D)
        k = _norm_rotate(s["qkv"][:, hq:hq + hkv], s["kn"], rope)
        _write(s, k[:, None], s["qkv"][:, hq + hkv:][:, None])
        return _read(s, s["dtype"]) + [q]
    if s["op"] == "read_back":
        return _read(s, s["dtype"])
    return _attend(s)


# ------------------------------------------------------- from the definition --
def _stored(x, fmt):
    """The values that vectors x (64 bits) read back as, in 64 bits."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == INT8:
        d = torch.clamp((amax / 127).float(), min=TINY).double()
        return torch.round(x / d) * d
    d = torch.exp2(torch.clamp(torch.ceil(torch.log2(amax / 448)), min=-126.0))
    d = torch.where(amax <= 448 * d / 2, d / 2, d).clamp(min=TINY)
    y = x / d
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))), min=-6.0) - 3)
    return torch.round(y / step) * step * d


def _tile_values(s, layer, seq, t0, t1):
    """K and V of tokens [t0, t1) of a sequence, [2][kv heads][tokens][128] in 64 bits."""
    t = torch.arange(t0, t1, device="cuda")
    tile = s["pool"][layer, s["table"][seq].long()[t // PAGE]]             # [tokens][heads][4224]
    got = []
    for part in (0, 1):
        at = (part * PAGE + t % PAGE)[:, None]
        raw = tile.gather(2, (at * D + torch.arange(D, device="cuda"))[:, None].expand(-1, s["hkv"], -1))
        d = tile.gather(2, (2 * PAGE * D + at * 4 + torch.arange(4, device="cuda"))[:, None].expand(-1, s["hkv"], -1))
        if s["fmt"] == INT8:
            x = raw.double()
            x = torch.where(x > 127, x - 256, x)
        else:
            b = raw.double()
            sign = torch.where(b > 127, -1.0, 1.0).double()
            b = torch.where(b > 127, b - 128, b)
            e, f = torch.floor(b / 8), b % 8
            x = sign * torch.where(e > 0, (8 + f) * torch.exp2(e - 10), f * 2.0 ** -9)
        got.append((x * d.contiguous().view(torch.float32).double()).transpose(0, 1))
    return torch.stack(got)


def exact(case, seed):
    s = prepare(case, seed)
    fmt, hq, hkv, lens, before = s["fmt"], s["hq"], s["hkv"], s["lens"], s["before"]
    if s["op"] == "append":
        return [_stored(s[x].double(), fmt).permute(1, 2, 0, 3).contiguous() for x in ("k", "v")]
    if s["op"] == "norm_append":
        x = s["qkv"].double()
        z = torch.view_as_complex(s["rope"].double())[s["pos"].long()][:, None]
        turned = []
        for part, w in ((x[:, :hq], s["qn"]), (x[:, hq:hq + hkv], s["kn"])):
            y = part * (part.square().sum(-1, keepdim=True) / D + EPS).rsqrt() * w.double()
            y = torch.complex(y[..., :64], y[..., 64:]) * z
            turned.append(torch.cat([y.real, y.imag], -1))
        kv = [_stored(y, fmt).transpose(0, 1)[None].contiguous() for y in (turned[1], x[:, hq + hkv:])]
        return kv + [turned[0] * D ** -0.5]
    if s["op"] == "read_back":
        got = [torch.cat([_tile_values(s, layer, i, before, before + m) for i, m in enumerate(lens)], 2)
               for layer in range(s["layers"])]
        return [torch.stack([x[part] for x in got]) for part in (0, 1)]
    out, row = [], 0
    for i, m in enumerate(lens):
        k, v = _tile_values(s, 0, i, 0, before + m)
        rows = 1 if s["op"] == "decode" else m
        o = []
        for h in range(hq):
            score = s["q"][row:row + rows, h].double() @ k[h * hkv // hq].T
            if rows > 1:
                score += torch.full_like(score, -torch.inf).triu(before + 1)
            o.append(torch.softmax(score, -1) @ v[h * hkv // hq])
        out.append(torch.stack(o, 1).reshape(rows, hq * D))
        row += rows
    return [torch.cat(out)]
