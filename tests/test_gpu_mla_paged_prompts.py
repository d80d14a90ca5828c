"""MLA.forward_paged of more than 64 tokens a sequence, on pages that there are not, counts out of range and rows that are not finite: against binary64 and
against the same tokens in pieces of 64, which take the form that reads the codes."""
import pytest
import torch

from test_gpu_mla import M, small_mla_params  # noqa: F401  (M: a fixture)
from test_gpu_mla_attention import C, NOPE, ROPE, V, _freqs, _layer

pytestmark = pytest.mark.gpu

DIM, HEADS, RANK = 256, 4, 128


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _case(M, seed, b, s, page, width, starts):
    """A layer, a cache whose rows in front of `starts` are written, a table of pages in no order, new tokens and their rotations."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, seed), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(seed)
    cache = LatentPages(b * width, page, device="cuda")
    table = torch.randperm(b * width, generator=g).view(b, width).int().cuda()
    turns = _freqs(ROPE, 2048).cuda()
    most = max(1, *starts)
    x = torch.randn(b, most + s, DIM, generator=g).bfloat16().cuda()
    freqs = turns[torch.arange(most)].expand(b, -1, -1).contiguous()
    with torch.inference_mode():
        layer.forward_paged(x[:, :most].contiguous(), cache, table, _ints(*[0] * b), _ints(*(max(0, n) for n in starts)), freqs, min(most, page * width))
    at = torch.tensor([[max(0, n) + i for i in range(s)] for n in starts])
    return layer, cache, table, x[:, most:].contiguous(), turns[at.cuda()].contiguous()


def _copy(cache):
    from dsv3fp8.model import LatentPages
    new = LatentPages(*cache.scale.shape, device="cuda")
    for mine, theirs in ((new.kv.view(torch.uint8), cache.kv.view(torch.uint8)), (new.scale, cache.scale), (new.pe, cache.pe)):
        mine.copy_(theirs)
    return new


def _reference(layer, x, cache, table, starts, counts, freqs, positions):
    """On a copy of the cache with the new rows written by the operator: the attention of the positions in a page in binary64; zeros for tokens that
    see none or that a sequence does not have."""
    from dsv3fp8 import kernel, model
    cache, (pages, page) = _copy(cache), cache.scale.shape
    layer.stack_a()
    qq, qs = torch.ops.dsv3fp8.mla_latent_paged(model.linear(x, layer._wa), layer.q_norm.weight, layer.kv_norm.weight, freqs, cache.kv, cache.scale, cache.pe,
                                                table, starts, counts, layer.q_norm.eps, layer.kv_norm.eps)
    kv, pe = cache.read(table, _ints(*[positions] * x.size(0)), positions)
    q = kernel.fp8_gemm(qq, qs, layer.wq_b.weight, layer.wq_b.scale).unflatten(-1, (HEADS, NOPE + ROPE)).double()
    w = kernel.weight_dequant(layer.wkv_b.weight, layer.wkv_b.scale).double().view(HEADS, NOPE + V, C)
    wo = kernel.weight_dequant(layer.wo.weight, layer.wo.scale).double()
    turn = torch.view_as_complex(q[..., NOPE:].unflatten(-1, (-1, 2)).contiguous()) * freqs.to(torch.complex128).unsqueeze(2)
    rope = torch.view_as_real(turn).flatten(3).bfloat16().double()
    out = torch.zeros(x.size(0), x.size(1), DIM, dtype=torch.float64, device="cuda")
    for i, (first, n) in enumerate(zip(starts.tolist(), counts.tolist())):
        entry = table[i].long()[torch.arange(positions, device="cuda") // page]
        there = ((entry >= 0) & (entry < pages)).nonzero().flatten()
        for t in range(min(n, x.size(1)) if first >= 0 else 0):
            use = there[there <= first + t]
            if use.numel():
                c, k = kv[i, use].double(), pe[i, use].double()
                heads = []
                for h in range(HEADS):
                    score = (c @ (q[i, t, h, :NOPE] @ w[h, :NOPE]) + k @ rope[i, t, h]) * layer.softmax_scale
                    heads.append(w[h, NOPE:] @ (score.softmax(0) @ c))
                out[i, t] = wo @ torch.cat(heads)
    return out


def _both(layer, x, cache, table, starts, counts, freqs, positions):
    """The prompt at once, and in pieces of 64 on a copy of the cache."""
    other, s, parts = _copy(cache), x.size(1), []
    with torch.inference_mode():
        y = layer.forward_paged(x, cache, table, starts, counts, freqs, positions)
        for k in range(0, s, 64):
            n = min(64, s - k)
            here = counts.long().sub(k).clamp(0, n).int()
            parts.append(layer.forward_paged(x[:, k:k + n].contiguous(), other, table, torch.where(starts < 0, starts, (starts.long() + k).clamp(max=2 ** 31 - 1).int()), here,
                                             freqs[:, k:k + n].contiguous(), positions))
    for a, c in ((cache.kv.view(torch.uint8), other.kv.view(torch.uint8)), (cache.scale.view(torch.int32), other.scale.view(torch.int32)),
                 (cache.pe.view(torch.int16), other.pe.view(torch.int16))):
        assert torch.equal(a, c)
    return y, torch.cat(parts, 1)


def _check(y, ref):
    # wo's input is off by half a step of e4m3 an element (2^-4 of it) and by the attention's 2^-7 of the norm; a random product carries both over in proportion;
    # the result rounds to bf16 (2^-8); keys, values, exponentials and scores of the explicit form round to bf16 as well, 2^-8 each.  Rows of zeros are zeros.
    assert ((y.double() - ref).norm(dim=-1) <= (2.0 ** -4 + 2.0 ** -7 + 5 * 2.0 ** -8) * ref.norm(dim=-1)).all()


@pytest.mark.parametrize("s,page,starts", [(70, 24, (50, 0, 7)), (65, 8, (0, 33, 64)), (130, 64, (100, 64, 0)), (200, 16, (0, 0, 90))])
def test_prompts_over_pages_that_there_are_not(M, s, page, starts):
    """Every second page is missing, in the prefix and under the new rows; the last sequence has none in front of its middle, so that its first tokens see nothing; the
    first has its first page only."""
    width = -(-(max(starts) + s) // page) + 1
    layer, cache, table, x, freqs = _case(M, s, 3, s, page, width, starts)
    holes = torch.tensor([-1, table.numel(), 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda").repeat(width)
    table[0, 1:], table[1, ::2], table[2, :width // 2], table[2, -2] = holes[:width - 1], holes[:(width + 1) // 2], holes[:width // 2], -5
    positions = max(starts) + s
    args = (layer, x, cache, table, _ints(*starts), _ints(s, s, s - 3), freqs, positions)
    ref = _reference(*args)
    nothing = (ref == 0).all(-1)
    assert nothing[2, :s - 3].any() == (starts[2] < width // 2 * page) and nothing[2, s - 3:].all()
    for y in _both(*args):
        assert torch.isfinite(y).all() and (y[nothing] == 0).all()
        _check(y, ref)


@pytest.mark.parametrize("what", ["token", "latent", "nan key", "inf key"])
def test_rows_that_are_not_finite_reach_the_tokens_that_see_them(M, what):
    """A new token of NaN in the middle of a block; rows of the prefix and of other sequences' pages likewise.  The others get the bits that they get without."""
    s, starts = 130, (40, 0, 100)
    layer, cache, table, x, freqs = _case(M, 7, 3, s, 24, 10, starts)
    args = (table, _ints(*starts), _ints(s, s, 90), freqs, 230)
    with torch.inference_mode():
        clean = layer.forward_paged(x, _copy(cache), *args)
    bad = [(0, 40 + 37), (1, 101)] if what == "token" else [(0, 33), (2, 99)]          # sequence, position
    for i, at in bad:
        row = int(table[i, at // 24]), at % 24
        if what == "token":
            x[i, at - starts[i], 5] = float("nan")
        elif what == "latent":
            cache.kv.view(torch.uint8)[row], cache.scale[row] = 0, float("nan")
        else:
            cache.pe[row][3] = float("nan" if what == "nan key" else "inf")
    nan = torch.zeros(3, s, dtype=torch.bool, device="cuda")
    for i, at in bad:
        nan[i, max(0, at - starts[i]):] = True
    nan[2, 90:] = False
    for n, y in enumerate(_both(layer, x, cache, *args)):
        if n == 0:
            assert torch.isnan(y[nan]).all() and torch.equal(y[~nan].view(torch.int16), clean[~nan].view(torch.int16))
        else:
            assert torch.isfinite(y[~nan]).all()
            assert what == "inf key" or torch.isnan(y[nan]).all()


def test_rows_behind_a_sequence_reach_nobody(M):
    """NaN in codes, scales and keys of all that no sequence has, as a page leaves them whose owner was another; fewer tokens than the widest sequence's."""
    s, starts = 70, (30, 0, 65)
    layer, cache, table, x, freqs = _case(M, 9, 3, s, 16, 10, starts)
    counts = (s, 66, 5)
    args = (table, _ints(*starts), _ints(*counts), freqs, 150)
    with torch.inference_mode():
        clean = layer.forward_paged(x, _copy(cache), *args)
    used = torch.zeros(*cache.scale.shape, dtype=torch.bool, device="cuda")
    for i, n in enumerate(starts):
        for at in range(n + counts[i]):
            used[int(table[i, at // 16]), at % 16] = True
    cache.kv.view(torch.uint8)[~used], cache.scale[~used], cache.pe[~used] = 0x7f, float("nan"), float("nan")
    for i, n in enumerate(counts):
        x[i, n:] = float("nan")
    y, pieces = _both(layer, x, cache, *args)
    assert torch.equal(y.view(torch.int16), clean.view(torch.int16)) and torch.isfinite(pieces).all()


def test_starts_and_counts_out_of_range(M):
    """Counts above the rows are all rows, negative ones and those of a negative start none; a start behind the stated positions sees these and writes nothing."""
    s, starts = 70, (60, 0, 5, 44)
    layer, cache, table, x, freqs = _case(M, 11, 4, s, 24, 6, starts)
    most = 2 ** 31 - 1
    with torch.inference_mode():
        want = layer.forward_paged(x, _copy(cache), table, _ints(*starts), _ints(s, s, s, s), freqs, 140)
    y, pieces = _both(layer, x, cache, table, _ints(60, 0, 5, -1), _ints(most, s + 1, -most - 1, s), freqs, 140)
    assert torch.equal(y[:2].view(torch.int16), want[:2].view(torch.int16)) and (y[2:] == 0).all()
    assert torch.isfinite(pieces).all() and (pieces[2:] == 0).all()
    args = (layer, x, cache, table, _ints(most, most - 69, most - 1, 44), _ints(s, s, most, s), freqs, 44)
    ref = _reference(*args)
    for got in _both(*args):
        _check(got, ref)


def test_a_prompt_captured_and_replayed(M):
    """One graph of a prompt's step, replayed after lengths, tables, inputs and rows that are not finite have changed on the device."""
    s = 70
    layer, cache, table, x, freqs = _case(M, 13, 2, s, 16, 9, (60, 20))
    start_cache, g = _copy(cache), torch.Generator().manual_seed(3)
    starts, counts = _ints(60, 20), _ints(s, s)
    with torch.inference_mode():
        layer.forward_paged(x, _copy(cache), table, starts, counts, freqs, 140)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward_paged(x, cache, table, starts, counts, freqs, 140)
        for step in range(6):
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
            if step % 2:
                x[0, 33, 5] = float("nan")
            starts.copy_(_ints(60 - 7 * step, 20 + step))
            counts.copy_(_ints(s - step, s))
            table.copy_(torch.randperm(18, generator=g).view(2, 9).int())
            if step > 2:
                table[1, step - 3] = -1
            for mine, theirs in ((cache.kv.view(torch.uint8), start_cache.kv.view(torch.uint8)), (cache.scale, start_cache.scale), (cache.pe, start_cache.pe)):
                mine.copy_(theirs)
            other = _copy(cache)
            graph.replay()
            want = layer.forward_paged(x, other, table, starts, counts, freqs, 140)
            torch.cuda.synchronize()
            for a, c in ((y, want), (cache.pe, other.pe)):
                assert torch.equal(a.view(torch.int16), c.view(torch.int16))
            assert torch.isnan(want[0, 33:s - step]).all() == bool(step % 2) and torch.isfinite(want[0, :33]).all()
