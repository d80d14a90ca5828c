"""MLA.forward_paged: prompts, single tokens, trees of drafted tokens and accepted paths of sequences of different lengths on one cache in pages."""
import pytest
import torch

from test_gpu_mla import M, small_mla_params  # noqa: F401  (M: a fixture)
from test_gpu_mla_attention import C, NOPE, ROPE, V, _freqs, _layer

pytestmark = pytest.mark.gpu

DIM, HEADS, RANK = 256, 4, 128


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tokens(g, b, s, at):
    """Inputs of b sequences' new tokens and the rotations of the positions `at` [b][s]."""
    return torch.randn(b, s, DIM, generator=g).bfloat16().cuda(), _freqs(ROPE, 512)[torch.tensor(at)].cuda()


def _reference(layer, x, cache, table, starts, counts, freqs, positions, seen):
    """Rows behind `starts` written by the operator into copies of the cache, the attention of the rows read back in binary64, without the
    quantisation in front of wo.  seen(i, t): the new tokens that token t of sequence i sees."""
    from dsv3fp8 import kernel, model
    pools = [t.clone() for t in (cache.kv, cache.scale, cache.pe)]
    layer.stack_a()
    qq, qs = torch.ops.dsv3fp8.mla_latent_paged(model.linear(x, layer._wa), layer.q_norm.weight, layer.kv_norm.weight, freqs, *pools, table, starts, counts,
                                                layer.q_norm.eps, layer.kv_norm.eps)
    kv, pe = torch.ops.dsv3fp8.mla_cache_read(*pools, table, starts + counts, positions)
    q = kernel.fp8_gemm(qq, qs, layer.wq_b.weight, layer.wq_b.scale).unflatten(-1, (HEADS, NOPE + ROPE)).double()
    w = kernel.weight_dequant(layer.wkv_b.weight, layer.wkv_b.scale).double().view(HEADS, NOPE + V, C)
    wo = kernel.weight_dequant(layer.wo.weight, layer.wo.scale).double()
    turn = torch.view_as_complex(q[..., NOPE:].unflatten(-1, (-1, 2)).contiguous()) * freqs.to(torch.complex128).unsqueeze(2)
    rope = torch.view_as_real(turn).flatten(3).bfloat16().double()
    out = torch.zeros(x.size(0), x.size(1), DIM, dtype=torch.float64, device="cuda")
    for i in range(x.size(0)):
        first = int(starts[i])
        for t in range(int(counts[i])):
            use = torch.tensor(list(range(first)) + [first + j for j in sorted(seen(i, t))], dtype=torch.long, device="cuda")
            c, k, heads = kv[i, use].double(), pe[i, use].double(), []
            for h in range(HEADS):
                score = (c @ (q[i, t, h, :NOPE] @ w[h, :NOPE]) + k @ rope[i, t, h]) * layer.softmax_scale
                heads.append(w[h, NOPE:] @ (score.softmax(0) @ c))
            out[i, t] = wo @ torch.cat(heads)
    return out


def _check(y, ref, counts):
    # wo's input is off by half a step of e4m3 an element (2^-4 of it; the smallest elements' 2^-10 of the block's scale is nothing beside that) and
    # by the attention's 2^-7 of the norm; a random product carries both over in proportion; the result rounds to bf16 (2^-8).
    # More than 64 tokens: keys, values, exponentials and scores of the explicit form round to bf16 as well, 2^-8 each
    assert ((y.double() - ref).norm(dim=-1) <= (2.0 ** -4 + 2.0 ** -7 + 5 * 2.0 ** -8) * ref.norm(dim=-1)).all()
    for i, n in enumerate(counts.tolist()):
        assert (y[i, n:] == 0).all()


def test_prompt_tokens_tree_and_accepted_path(M):
    """Three sequences of 70, 33 and no tokens; then a token each (the third's first); a tree of six; the accepted nodes kept; a token again."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 41), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(42)
    b, page, pages = 3, 24, 16
    cache = LatentPages(pages, page, device="cuda")
    table = torch.randperm(pages, generator=g)[:b * 5].view(b, 5).int().cuda()
    lengths = [0, 0, 0]

    def step(s, counts, depths, tree=None, seen=None):
        nonlocal lengths
        starts, counts = _ints(*lengths), _ints(*counts)
        x, freqs = _tokens(g, b, s, [[n + d for d in depths] for n in lengths])
        positions = max(lengths) + s
        ref = _reference(layer, x, cache, table, starts, counts, freqs, positions, seen or (lambda i, t: range(t + 1)))
        x[torch.arange(s, device="cuda") >= counts[:, None]] = float("nan")         # (tokens that a sequence does not have)
        with torch.inference_mode():
            y = layer.forward_paged(x, cache, table, starts, counts, freqs, positions, tree)
        assert y.shape == (b, s, DIM) and y.dtype == torch.bfloat16
        _check(y, ref, counts)
        return starts, counts

    _, counts = step(70, (70, 33, 0), range(70))
    lengths = [70, 33, 0]
    step(1, (1, 1, 1), [0])
    lengths = [n + 1 for n in lengths]
    # nodes 0 -> 1 -> 3 -> 5, 0 -> 2 -> 4
    parents, depths = [None, 0, 0, 1, 2, 3], [0, 1, 1, 2, 2, 3]
    sets = []
    for i, p in enumerate(parents):
        sets.append({i} | (sets[p] if p is not None else set()))
    tree = torch.tensor([[sum(1 << j for j in s) for s in sets]] * b).cuda()
    starts, _ = step(6, (6, 6, 3), depths, tree, lambda i, t: sets[t])
    before, _ = cache.read(table, _ints(*(n + 6 for n in lengths)), max(lengths) + 6)
    path, kept = torch.tensor([[0, 1, 3, 5], [0, 2, 4, 9], [0, 2, 9, 9]], dtype=torch.int32).cuda(), _ints(4, 3, 2)
    cache.keep(table, starts, path, kept)
    after, _ = cache.read(table, starts + kept, max(lengths) + 6)
    for i, nodes in enumerate(([0, 1, 3, 5], [0, 2, 4], [0, 2])):
        n = lengths[i]
        assert torch.equal(after[i, :n], before[i, :n]) and torch.equal(after[i, n:n + len(nodes)], before[i, [n + k for k in nodes]])
        assert (after[i, n + len(nodes):] == 0).all()
    lengths = [n + k for n, k in zip(lengths, (4, 3, 2))]
    step(1, (1, 0, 1), [0])


@pytest.mark.parametrize("s", [5, 70])
def test_paged_against_the_contiguous_cache(M, s):
    """The same steps on both caches: the rows differ by one quantisation to e4m3 (half a step, 2^-4 at most), the scores of these layers are small, and
    wo's input is quantised in both."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 43), DIM, HEADS, RANK, 96)
    g = torch.Generator().manual_seed(44)
    freqs = _freqs(ROPE, 96).cuda()
    cache = LatentPages(6, 32, device="cuda")
    table = torch.tensor([[4, 0, 3], [1, 5, 2]], dtype=torch.int32).cuda()
    at = 0
    for n in (s, 1):
        x = torch.randn(2, n, DIM, generator=g).bfloat16().cuda()
        mask = torch.full((n, n), float("-inf"), device="cuda").triu_(1) if n > 1 else None
        with torch.inference_mode():
            want = layer(x, at, freqs[at:at + n], mask)
            got = layer.forward_paged(x, cache, table, _ints(at, at), _ints(n, n), freqs[at:at + n].expand(2, -1, -1).contiguous(), at + n)
        # rows 2^-4, both inputs of wo 2^-4 each
        assert ((got.double() - want.double()).norm(dim=-1) <= 3 * 2.0 ** -4 * want.double().norm(dim=-1)).all()
        at += n
    kv, pe = cache.read(table, _ints(at, at), at)
    # norms and rotations may round to the neighbouring bf16 (2^-7), codes are off by half a step (2^-4, of the smallest 2^-10 of a scale below 2^-5)
    for a, c, steps, least in ((pe, layer.pe_cache, 2.0 ** -7, 2.0 ** -16), (kv, layer.kv_cache, 2.0 ** -4 + 2.0 ** -7, 2.0 ** -15)):
        assert ((a.double() - c[:, :at].double()).abs() <= steps * c[:, :at].double().abs() + least).all()


def test_a_captured_step_serves_every_length(M):
    """One graph of a decode step, replayed after lengths, page table and inputs have changed on the device."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 45), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(46)
    cache, other = LatentPages(8, 16, device="cuda"), LatentPages(8, 16, device="cuda")
    table = torch.tensor([[2, 7, 1], [0, 4, 5]], dtype=torch.int32).cuda()
    x, freqs = _tokens(g, 2, 1, [[0], [0]])
    starts, counts = _ints(0, 0), _ints(1, 1)
    with torch.inference_mode():
        layer.forward_paged(x, other, table, starts, counts, freqs, 48)
        for mine, warm in ((cache.kv.view(torch.uint8), other.kv.view(torch.uint8)), (cache.scale, other.scale), (cache.pe, other.pe)):
            mine.copy_(warm)            # (position 0 of the second sequence, which the first step leaves as it is)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward_paged(x, cache, table, starts, counts, freqs, 48)
        for step in range(40):
            new, turn = _tokens(g, 2, 1, [[step], [step]])
            x.copy_(new)
            freqs.copy_(turn)
            starts.fill_(step)
            counts.copy_(_ints(1, step % 2))
            graph.replay()
            want = layer.forward_paged(new, other, table, starts, counts, turn, 48)
            torch.cuda.synchronize()
            assert torch.equal(y.view(torch.int16), want.view(torch.int16))
    for a, c in ((cache.kv.view(torch.uint8), other.kv.view(torch.uint8)), (cache.scale, other.scale), (cache.pe, other.pe)):
        assert torch.equal(a, c)
