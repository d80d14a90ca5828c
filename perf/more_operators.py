"""Operators on microscaled 4-bit numbers, and what is timed of them: tensors turned into them and back, the linear layers' product with
weights held so, and the attention layer's latent cache in pages of 4-bit rows, written, read back and attended to.

The format: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), two to a byte, the even one in the low half, and for every 32
of them along the last dimension one power of two in a byte of its own (e8m0: 2^(byte - 127), 255 is NaN).  Codes are held as
``torch.float4_e2m1fn_x2``, scales as ``torch.float8_e8m0fnu``.

Four paths:
  convert  ``mx4_quant`` and ``mx4_dequant``: into four bits and back, what a calibration run or a checkpoint's conversion looks at
  product  ``mx4_gemm``: a weight of four bits, activations of four bits or e4m3 ones with a power of two per 128
  store    ``mla_latent_paged`` and ``mla_cache_read`` on pages of 4-bit rows: a step's new rows written, the prefix read back
  attend   ``mla_decode_paged`` on such pages: one new token or a tree of drafted ones per sequence

A layer's cache is three arrays of pages that many sequences share: ``kv_pages`` e2m1 [pages, page, 256], ``kv_scale`` e8m0 [pages,
page, 16] and ``pe_pages`` bf16 [pages, page, 64].  ``page_table`` int32 [batch, width] names a sequence's pages in order (-1 where it
has none), ``starts`` its positions before this step and ``counts`` its new rows, which take the positions behind them.  In a
cache row no scale lies more than 2^14 below the row's largest.

Head dimensions are those of ``dsv3fp8.model.ModelArgs``; 128 heads are its own, 16 a rank's share of them.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False
FP8, FP4, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
DEVICE = "cuda"
C, ROPE, NOPE, V = 512, 64, 128, 128
SOFTMAX_SCALE = 192 ** -0.5 * (0.1 * math.log(40) + 1) ** 2       # with the extended window's correction
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_ELEMENTS = 18432 * 7168            # of the largest convert case
MOST_PRODUCTS = 4096 * 18432 * 7168     # of the largest product case
MOST_PAIRS = 61 * 128 * 32768           # (row, position) pairs of the largest attend case
MOST_POSITIONS = 64 * 8192              # cached positions of all sequences


# ------------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token's activations: only latency counts
        {"name": "convert_1x7168", "path": "convert", "rows": 1, "width": 7168, "type": "bf16"},
        # the largest weight of the configuration
        {"name": "convert_18432x7168", "path": "convert", "rows": 18432, "width": 7168, "type": "bf16"},
        # one token through a projection: the weight is what has to be read
        {"name": "product_1x7168x18432", "path": "product", "m": 1, "k": 7168, "n": 18432, "act": "e4m3"},
        # a decode batch through the output projection
        {"name": "product_32x16384x7168", "path": "product", "m": 32, "k": 16384, "n": 7168, "act": "mx4"},
        # a short prompt, a row count that fills no tile
        {"name": "product_500x7168x4096", "path": "product", "m": 500, "k": 7168, "n": 4096, "act": "e4m3"},
        # a long prompt through a projection: bound by the matrix cores
        {"name": "product_4096x7168x18432", "path": "product", "m": 4096, "k": 7168, "n": 18432, "act": "mx4"},
        # a batch of drafted trees, some with fewer nodes than the widest
        {"name": "store_32x21", "path": "store", "batch": 32, "rows": 21, "q_rank": 1536, "page": 32},
        # a prompt of a layer without a low-rank query
        {"name": "store_1x4000", "path": "store", "batch": 1, "rows": 4000, "q_rank": 0, "page": 64},
        # one sequence early in its answer
        {"name": "decode_1x700", "path": "attend", "batch": 1, "nodes": 1, "context": 700, "heads": 128, "page": 64},
        # one rank's heads of a wide batch: the cache itself is what has to be read
        {"name": "decode_64x8192_h16", "path": "attend", "batch": 64, "nodes": 1, "context": 8192, "heads": 16, "page": 32},
        # drafted trees of a small batch, pages that end inside a tile
        {"name": "tree_8x25x2001", "path": "attend", "batch": 8, "nodes": 25, "context": 2001, "heads": 128, "page": 24},
        # one long context with a wide draft
        {"name": "tree_1x61x32768", "path": "attend", "batch": 1, "nodes": 61, "context": 32768, "heads": 128, "page": 128},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(["convert", "convert", "product", "product", "product", "product", "store", "store", "attend", "attend", "attend"])
    if path == "convert":
        width = 32 * _log_int(rng, 1, 576)
        return {"path": path, "rows": _log_int(rng, 1, min(MOST_ELEMENTS // width, 65536)), "width": width, "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if path == "product":
        m, k = _log_int(rng, 1, 4096), 128 * _log_int(rng, 1, 144)
        n = _log_int(rng, 1, 24576)
        return {"path": path, "m": m, "k": k, "n": min(n, MOST_PRODUCTS // (m * k)), "act": rng.choice(["e4m3", "mx4"])}
    page = 8 * _log_int(rng, 1, 32)
    if path == "store":
        batch = _log_int(rng, 1, 64)
        return {"path": path, "batch": batch, "rows": _log_int(rng, 1, 4000 // batch), "q_rank": rng.choice([0, 512, 1536]), "page": page}
    batch, nodes = _log_int(rng, 1, 64), rng.choice([1, _log_int(rng, 2, 64)])
    heads = rng.choice([4, 16, 20, 64, 128])
    most = min(MOST_PAIRS // (batch * nodes * heads), MOST_POSITIONS // batch, 32768)
    return {"path": path, "batch": batch, "nodes": nodes, "context": _log_int(rng, nodes, max(nodes, most)), "heads": heads, "page": page}


# -------------------------------------------------------------------------------- the format, in elementary operations

def _values_of_codes():
    magnitudes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEVICE)
    one = torch.cat([magnitudes, -magnitudes])
    byte = torch.arange(256, device=DEVICE)
    return torch.stack((one[byte & 15], one[byte >> 4]), -1)          # of the two codes of a byte


def _power(byte):
    """2^(byte - 127) in binary32, NaN for 255."""
    p = torch.ldexp(torch.ones(byte.shape, device=byte.device), byte.int() - 127)
    return torch.where(byte == 255, float("nan"), p)


def _unpacked(codes, scale):
    """Values in binary32 of packed codes [.., n / 2] and scales [.., n / 32]."""
    values = _values_of_codes()[codes.view(torch.uint8).int()].flatten(-2)
    return (values.unflatten(-1, (-1, 32)) * _power(scale.view(torch.uint8))[..., None]).flatten(-2)


def _scale_bytes(x):
    """Of blocks [.., n / 32, 32] in binary32: the smallest power of two that no element is more than six times of."""
    top = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)                              # top = mantissa 2^exponent, mantissa in [1/2, 1)
    byte = (exponent - 3 + (mantissa > 0.75).int() + 127).clamp(0, 254)
    byte = torch.where(top > 0, byte, 0)
    return torch.where(top < float("inf"), byte, 255)


def _codes(x, byte):
    """e2m1 codes, ties to the even one, of blocks [.., n / 32, 32] in binary32 with these scales, packed; zeros where the scale is NaN."""
    x = torch.ldexp(x, 127 - byte.int()[..., None])
    a = x.abs()
    # the midpoints between neighbouring magnitudes, each counted where it goes up: to the magnitude whose code is even
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = (code | (torch.signbit(x).int() << 3)).masked_fill(byte[..., None] == 255, 0).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4


def _packed(x, row=False):
    """Codes and scales, as bytes; `row`: none of a row's scales more than 2^14 below its largest, and all NaN if one is."""
    blocks = x.float().unflatten(-1, (-1, 32))
    byte = _scale_bytes(blocks)
    if row:
        top = byte.amax(-1, keepdim=True)
        byte = torch.where(top == 255, 255, torch.maximum(byte, top - 14))
    return _codes(blocks, byte), byte.to(torch.uint8)


# ------------------------------------------------------------------------------------------------------- preparation

def _lengths(rng, batch, longest, least):
    """Positions of the sequences, this step's included: spread over a factor of eight, the first the longest."""
    lo = max(least, longest // 8, 1)
    return [longest] + [_log_int(rng, lo, max(lo, longest)) for _ in range(batch - 1)]


def _cache(rng, g, lengths, longest, page):
    """A cache with rows in every page and room for sequences of the longest length, and their tables: pages in no order, -1 behind
    the last."""
    need, most = [-(-n // page) for n in lengths], -(-longest // page)
    pages = len(lengths) * most + 2
    # a latent's elements are of different sizes, as a norm's weight leaves them
    sizes = torch.exp(0.5 * torch.randn(C, generator=g, device=DEVICE))
    codes, scale = [], []
    for rows in torch.arange(pages * page).split(1 << 18):             # (a few at a time: the formation takes many times the rows' size)
        x = (torch.randn(rows.numel(), C, generator=g, device=DEVICE) * sizes).bfloat16()
        c, s = _packed(x, row=True)
        codes.append(c)
        scale.append(s)
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.full((len(lengths), most + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return {"kv": torch.cat(codes).view(pages, page, C // 2).view(FP4), "scale": torch.cat(scale).view(pages, page, C // 32).view(E8M0),
            "pe": torch.randn(pages, page, ROPE, generator=g, device=DEVICE).bfloat16(), "table": table.to(DEVICE)}


def _phases(g, *shape):
    angle = torch.rand(*shape, ROPE // 2, generator=g, device=DEVICE) * (2 * math.pi)
    return torch.polar(torch.ones_like(angle), angle)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _tree(rng, counts, nodes):
    """Ancestors and self of every node as bits; nodes that a sequence does not have see nothing."""
    rows = []
    for n in counts:
        bits = []
        for i in range(n):
            bits.append((bits[rng.randrange(max(0, i - 6), i)] if i else 0) | 1 << i)
        rows.append([v - (1 << 64) if v >> 63 else v for v in bits] + [0] * (nodes - n))
    return _ints(rows, torch.int64)


def _activations(g, rows, width, dtype=torch.bfloat16):
    """Tokens of different sizes, and a few channels that are larger than the rest in all of them."""
    x = torch.randn(rows, width, generator=g, device=DEVICE) * torch.exp(torch.randn(rows, 1, generator=g, device=DEVICE))
    x[:, ::97] *= 8
    return x.to(dtype)


def prepare(case, seed):
    rng, g = random.Random(seed), torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    path = case["path"]
    if path == "convert":
        state = {"x": _activations(g, case["rows"], case["width"], TYPES[case["type"]])}
    elif path == "product":
        m, n, k = case["m"], case["n"], case["k"]
        x = _activations(g, m, k).float()
        if case["act"] == "mx4":
            a, a_s = _packed(x)
            a, a_s = a.view(FP4), a_s.view(E8M0)
        else:
            a, a_s = _quantised(x.unflatten(-1, (-1, 128)))
            a = a.flatten(-2)
        b, b_s = _packed(torch.randn(n, k, generator=g, device=DEVICE) * 0.02)
        state = {"a": a, "a_s": a_s, "b": b.view(FP4), "b_s": b_s.view(E8M0)}
    elif path == "store":
        batch, rows, rank, page = case["batch"], case["rows"], case["q_rank"], case["page"]
        counts = [rows] + [rng.randint(-(-rows // 2), rows) for _ in range(batch - 1)]
        starts = [rng.randrange(0, 100) for _ in range(batch)]
        ends = [s + n for s, n in zip(starts, counts)]
        state = _cache(rng, g, ends, 100 + rows, page)
        state |= {"a": torch.randn(batch, rows, rank + C + ROPE, generator=g, device=DEVICE).bfloat16(),
                  "q_norm": (1 + 0.1 * torch.randn(rank, generator=g, device=DEVICE)).bfloat16() if rank else None,
                  "kv_norm": torch.exp(0.5 * torch.randn(C, generator=g, device=DEVICE)).bfloat16(),
                  "freqs": _phases(g, batch, rows), "starts": _ints(starts), "counts": _ints(counts), "lengths": _ints(ends),
                  "positions": 100 + rows}
    else:
        batch, nodes, heads, page = case["batch"], case["nodes"], case["heads"], case["page"]
        lengths = _lengths(rng, batch, case["context"], nodes)
        counts = [nodes] + [rng.randint(-(-nodes // 2), nodes) for _ in range(batch - 1)]
        state = _cache(rng, g, lengths, case["context"], page)
        w = torch.randn(heads * 2, 128, C // 128, 128, generator=g, device=DEVICE) * 0.02
        w_scale = (w.abs().amax((1, 3)) / 448).float()
        state |= {"q": torch.randn(batch, nodes, heads, NOPE + ROPE, generator=g, device=DEVICE).bfloat16(),
                  "freqs": _phases(g, batch, nodes), "starts": _ints([n - c for n, c in zip(lengths, counts)]), "counts": _ints(counts),
                  "tree": _tree(rng, counts, nodes) if nodes > 1 else None,
                  "w": (w / w_scale[:, None, :, None]).to(FP8).view(heads * (NOPE + V), C), "w_scale": w_scale,
                  "positions": case["context"]}
    state["path"] = path
    return state


# -------------------------------------------------------------------------------------------------------- plain forms

def _block_scale(x):
    top = x.abs().amax(-1).clamp_min(1e-4)
    return top / torch.full_like(top, 448.0)        # (a plain number would be multiplied with as its reciprocal)


def _quantised(x):
    """e4m3 codes and one power of two for each of the last dimension's runs."""
    s = _block_scale(x)
    mantissa, exponent = torch.frexp(s)
    s = torch.ldexp(torch.ones_like(s), exponent - (mantissa == 0.5).int())
    return (x / s[..., None]).to(FP8), s


def _convert(state):
    return _unpacked(*_packed(state["x"])).bfloat16()


def _product(state):
    a = state["a"]
    if a.dtype == FP4:
        x = _unpacked(a, state["a_s"])
    else:
        x = (a.float().unflatten(-1, (-1, 128)) * state["a_s"][..., None]).flatten(-2)
    return torch.matmul(x, _unpacked(state["b"], state["b_s"]).t()).bfloat16()


def _normed(x, w):
    """The root in 64 bits: a sum's last bit would decide roundings behind it."""
    x64 = x.double()
    r = (1 / (x64 * x64).mean(-1, keepdim=True).add(EPS).sqrt()).float()
    return (x.float() * r * w.float()).bfloat16()


def _rotated(x, freqs):
    re, im = x.float().unflatten(-1, (-1, 2)).unbind(-1)
    cos, sin = freqs.real, freqs.imag
    return torch.stack((re * cos - im * sin, re * sin + im * cos), -1).flatten(-2)


def _rows(state, positions):
    """Cache rows [batch, ..] of the sequences' positions; those of positions without a page name a row, any."""
    page, table = state["kv"].size(1), state["table"]
    entry = table.gather(1, (positions // page).clamp(0, table.size(1) - 1))
    return entry.clamp_min(0).long() * page + positions % page


def _latents(state, rows):
    codes, scale = state["kv"].view(torch.uint8).view(-1, C // 2)[rows], state["scale"].view(torch.uint8).view(-1, C // 32)[rows]
    return _unpacked(codes, scale)


def _store(state):
    a, counts = state["a"], state["counts"]
    rank = a.size(2) - C - ROPE
    y, ys = a.new_empty(*a.shape[:2], 0, dtype=FP8), a.new_empty(*a.shape[:2], 0, dtype=torch.float32)
    if rank:
        n = _normed(a[..., :rank], state["q_norm"]).float().unflatten(-1, (-1, 128))
        ys = _block_scale(n)
        y = (n / ys[..., None]).to(FP8).flatten(-2)
    codes, scale = _packed(_normed(a[..., rank:rank + C], state["kv_norm"]), row=True)
    pe = _rotated(a[..., rank + C:], state["freqs"]).bfloat16()
    i = torch.arange(a.size(1), device=a.device)
    rows = _rows(state, (state["starts"][:, None] + i).long())
    live = (i < counts[:, None]).nonzero(as_tuple=True)
    rows = rows[live]
    state["kv"].view(torch.uint8).view(-1, C // 2)[rows] = codes[live]
    state["scale"].view(torch.uint8).view(-1, C // 32)[rows] = scale[live]
    state["pe"].view(-1, ROPE)[rows] = pe[live]
    # and back
    j = torch.arange(state["positions"], device=DEVICE).expand(counts.numel(), -1)
    rows = _rows(state, j)
    behind = (j >= state["lengths"][:, None])[..., None]
    return {"y": y, "ys": ys, "kv": _latents(state, rows).masked_fill(behind, 0).bfloat16(),
            "pe": state["pe"].view(-1, ROPE)[rows].masked_fill(behind, 0)}


def _visible(state, positions):
    """[batch, nodes, positions]: what each new token sees."""
    starts, counts = state["starts"].long()[:, None, None], state["counts"].long()[:, None, None]
    nodes = state["q"].size(1)
    i, j = torch.arange(nodes, device=DEVICE)[None, :, None], torch.arange(positions, device=DEVICE)[None, None]
    node = j - starts
    if state["tree"] is None:
        seen = node <= i
    else:
        seen = (node < 0) | (state["tree"][:, :, None] >> node.clamp(0, 63) & 1).bool()
    return seen & (node < counts) & (i < counts)


def _attend(state):
    q, positions = state["q"], state["positions"]
    batch, nodes, heads, _ = q.shape
    w = state["w"].float().view(heads * 2, 128, C // 128, 128) * state["w_scale"][:, None, :, None]
    w = w.bfloat16().float().view(heads, NOPE + V, C)           # the weight is a bf16 one, held in eight bits
    rows = _rows(state, torch.arange(positions, device=DEVICE).expand(batch, -1))
    latent, key = _latents(state, rows), state["pe"].view(-1, ROPE)[rows].float()
    q_pe = _rotated(q[..., NOPE:], state["freqs"][:, :, None])
    q_latent = torch.matmul(q[..., :NOPE].float().view(-1, heads, NOPE).transpose(0, 1).contiguous(), w[:, :NOPE])
    q_latent = q_latent.transpose(0, 1).reshape(batch, nodes * heads, C)
    scores = torch.matmul(q_latent, latent.transpose(1, 2).contiguous())
    scores += torch.matmul(q_pe.reshape(batch, nodes * heads, ROPE), key.transpose(1, 2).contiguous())
    seen = _visible(state, positions)
    scores = (scores * SOFTMAX_SCALE).view(batch, nodes, heads, positions).masked_fill_(~seen[:, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, nodes * heads, positions), latent).view(batch, nodes, heads, C)
    out = torch.where(total > 0, out / total, 0.0)
    out = torch.matmul(out.view(-1, heads, C).transpose(0, 1).contiguous(), w[:, NOPE:].transpose(1, 2).contiguous())
    return out.transpose(0, 1).reshape(batch, nodes, heads * V).bfloat16()


# -------------------------------------------------------------------------------------------------------- one pass

BF16 = 0            # the operators' code of a result's type


def _ops():
    """The framework's operators; a program imports it once."""
    if "dsv3fp8" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "deepseek-v3_amd"))      # the working folder is the tree to be measured
        import dsv3fp8  # noqa: F401
    return torch.ops.dsv3fp8


def _cache_args(s):
    return s["kv"], s["scale"], s["pe"], s["table"]


def run(state):
    with torch.inference_mode():
        path = state["path"]
        if own:
            ops = _ops()
            if path == "convert":
                return ops.mx4_dequant(*ops.mx4_quant(state["x"]), BF16)
            if path == "product":
                return ops.mx4_gemm(state["a"], state["a_s"], state["b"], state["b_s"], BF16)
            if path == "store":
                y, ys = ops.mla_latent_paged(state["a"], state["q_norm"], state["kv_norm"], state["freqs"], *_cache_args(state),
                                             state["starts"], state["counts"], EPS, EPS)
                kv, pe = ops.mla_cache_read(*_cache_args(state), state["lengths"], state["positions"])
                return {"y": y, "ys": ys, "kv": kv, "pe": pe}
            return ops.mla_decode_paged(state["q"], state["freqs"], *_cache_args(state), state["starts"], state["counts"], state["tree"],
                                        state["w"], state["w_scale"], state["positions"], SOFTMAX_SCALE)
        return {"convert": _convert, "product": _product, "store": _store, "attend": _attend}[path](state)


# ------------------------------------------------------------------------------------------- what a pass cannot avoid

def work(case):
    """Sequences whose length the seed draws count with the mean of their range's ends."""
    path = case["path"]
    if path == "convert":
        n = case["rows"] * case["width"]
        return {"bytes": n * ((4 if case["type"] == "f32" else 2) + 2), "flops": 2 * n}
    if path == "product":
        m, n, k = case["m"], case["n"], case["k"]
        act = k / 2 + k / 32 if case["act"] == "mx4" else k + k / 32
        return {"bytes": m * act + n * (k / 2 + k / 32) + 2 * m * n, "flops": 2 * m * n * k}
    row, batch = C // 2 + C // 32 + 2 * ROPE, case["batch"]
    if path == "store":
        rank, n = case["q_rank"], case["rows"] * (1 + 0.75 * (batch - 1))
        total = case["rows"] * batch
        return {"bytes": 2 * total * rank + n * (2 * (C + ROPE) + 4 * ROPE) + total * (rank + rank // 32) + batch * (100 + case["rows"]) * 2 * (C + ROPE) + n * row + 50 * batch * row,
                "flops": 4 * total * (rank + C)}
    nodes, heads = case["nodes"], case["heads"]
    total = case["context"] * (1 + (batch - 1) * 0.42)
    rows = nodes * heads * (1 + (batch - 1) * 0.75)
    return {"bytes": total * row + rows * 2 * (NOPE + ROPE + V) + heads * (NOPE + V) * C,
            "flops": 2 * rows * total / batch * (2 * C + ROPE) + 2 * rows * C * (NOPE + V)}


# ---------------------------------------------------------------------------------------------------------- in 64 bits

def _rounded(x, bits, least):
    """The nearest number of `bits` fraction bits, ties to even, whose exponent is at least `least`."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), e.clamp_min(least + 1) - 1 - bits)
    return (x / step).round() * step


def _bf16(x):
    return _rounded(x, 7, -126)


def _e2m1_64(x, cache_row=False):
    """The values that 4-bit numbers stand for: scales from logarithms, codes as numbers of one fraction bit down to 1."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, (top / 6).log2(), -127.0).ceil().clamp(-127, 127)
    e = torch.where(6 * torch.exp2(e - 1) >= top, (e - 1).clamp_min(-127), e)          # a logarithm may lie a bit too high
    if cache_row:
        e = torch.maximum(e, e.amax(-2, keepdim=True) - 14)
    s = torch.exp2(e)
    return (_rounded(blocks / s, 1, 0) * s).flatten(-2)


def _held(codes, scale):
    """The values of packed codes, bit by bit."""
    byte = codes.view(torch.uint8).long()
    code = torch.stack((byte & 15, byte >> 4), -1).flatten(-2)
    e, m = (code >> 1 & 3).double(), (code & 1).double()
    value = torch.where(e > 0, (1 + m / 2) * torch.exp2(e - 1), m / 2) * (1 - 2 * (code >> 3).double())
    return (value.unflatten(-1, (-1, 32)) * torch.exp2(scale.view(torch.uint8).double() - 127)[..., None]).flatten(-2)


def _norm64(x, w):
    return _bf16(x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w)


def _turn64(x, freqs):
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * freqs.to(torch.complex128)
    return torch.view_as_real(z).flatten(-2)


def _places(s, b, first, n):
    """Cache rows of n positions of sequence b from `first` on."""
    page, entries = s["kv"].size(1), s["table"][b].tolist()
    return [entries[j // page] * page + j % page for j in range(first, first + n)]


def exact(case, seed):
    s = prepare(case, seed)
    path = case["path"]
    if path == "convert":
        return torch.cat([_e2m1_64(x.double()) for x in s["x"].split(4096)])
    if path == "product":
        if case["act"] == "mx4":
            x = _held(s["a"], s["a_s"])
        else:
            x = s["a"].double() * s["a_s"].double().repeat_interleave(128, 1)
        return torch.cat([x @ _held(b, b_s).t() for b, b_s in zip(s["b"].view(torch.uint8).split(2048), s["b_s"].view(torch.uint8).split(2048))], 1)
    batch = case["batch"]
    codes, scale, pe = s["kv"].view(torch.uint8).view(-1, C // 2), s["scale"].view(torch.uint8).view(-1, C // 32), s["pe"].double().view(-1, ROPE)
    if path == "store":
        a, rank = s["a"].double(), case["q_rank"]
        y, ys = a.new_empty(*a.shape[:2], 0), a.new_empty(*a.shape[:2], 0)
        if rank:
            n = _norm64(a[..., :rank], s["q_norm"].double()).unflatten(-1, (-1, 128))
            ys = n.abs().amax(-1).clamp_min(1e-4) / 448
            y = _rounded(n / ys[..., None], 3, -6).flatten(-2)
        new = _e2m1_64(_norm64(a[..., rank:rank + C], s["kv_norm"].double()), cache_row=True)
        turned = _turn64(a[..., rank + C:], s["freqs"])
        kv, key = (torch.zeros(batch, s["positions"], n, dtype=torch.float64, device=DEVICE) for n in (C, ROPE))
        for b, (first, m) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
            at = torch.tensor(_places(s, b, 0, first), dtype=torch.long, device=DEVICE)
            kv[b, :first], key[b, :first] = _held(codes[at], scale[at]), pe[at]
            kv[b, first:first + m], key[b, first:first + m] = new[b, :m], turned[b, :m]
        return {"y": y, "ys": ys, "kv": kv, "pe": key}
    nodes, heads = case["nodes"], case["heads"]
    w = s["w"].double() * s["w_scale"].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    w = _bf16(w).view(heads, NOPE + V, C)
    out = torch.zeros(batch, nodes, heads, V, dtype=torch.float64, device=DEVICE)
    trees = s["tree"].tolist() if s["tree"] is not None else [[1]] * batch
    for b, (first, m) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
        at = torch.tensor(_places(s, b, 0, first + m), device=DEVICE)
        c, k, q = _held(codes[at], scale[at]), pe[at], s["q"][b, :m].double()
        turned = _turn64(q[..., NOPE:], s["freqs"][b, :m, None])
        hidden = torch.zeros(m, first + m, dtype=torch.bool)
        for i in range(m):
            for n in range(m):
                hidden[i, first + n] = not trees[b][i] >> n & 1
        hidden = hidden.to(DEVICE)
        for h in range(heads):
            score = ((q[:, h, :NOPE] @ w[h, :NOPE]) @ c.T + turned[:, h] @ k.T) * SOFTMAX_SCALE
            out[b, :m, h] = score.masked_fill(hidden, float("-inf")).softmax(-1) @ c @ w[h, NOPE:].T
    return out.view(batch, nodes, heads * V)
