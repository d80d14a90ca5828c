"""Layers of 4-bit weights, and MLA.forward_paged on pages of 4-bit rows: prompts, single tokens, trees of drafted tokens and accepted paths."""
import pytest
import torch
import torch.nn.functional as F

import test_gpu_mla_paged_layer as eight
from test_gpu_mla import M, small_mla_params  # noqa: F401  (M: a fixture)
from test_gpu_mla_attention import C, NOPE, ROPE, V, _freqs, _layer
from test_gpu_mla_paged_layer import DIM, HEADS, RANK, _check, _ints, _reference, _tokens

pytestmark = pytest.mark.gpu

FP8, FP4, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


@pytest.fixture
def four(M, monkeypatch):  # noqa: F811
    """The layers' weights are of four bits."""
    monkeypatch.setattr(M, "mx4_activations", "e4m3")
    M.Linear.dtype = FP4
    return M


def _fill(module, g):
    """Random weights in every linear layer; returns them as the numbers that they stand for, by name."""
    from dsv3fp8 import kernel
    values = {}
    for name, p in list(module.named_parameters()):
        if p.dtype == FP4:
            w = torch.randn(p.size(0), p.size(1) * 2, generator=g).mul_(0.05).bfloat16().cuda()
            codes, scale = kernel.mx4_quant(w)
            p.data, p.scale.data = codes, scale
            values[name] = kernel.mx4_dequant(codes, scale)
        elif not name.endswith("scale"):
            p.data.copy_(torch.randn(p.shape, generator=g).mul_(0.05).add_(1 if "norm" in name else 0))
    return values


@pytest.mark.parametrize("m", [1, 3, 40, 150])
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "mx4"])
def test_linear(four, monkeypatch, kind, m):
    """The composition of its operators, bit for bit, and near the product that it stands for: activations rounded to e4m3 are off by 2^-4 of themselves (the
    smallest by half of 2^-9 of a scale, which is below 2^-8 of the block's largest), to e2m1 by a quarter of themselves or of their scale, which is a third of
    the block's largest at most and more than a sixth."""
    from dsv3fp8 import kernel
    g = torch.Generator().manual_seed(m)
    if kind == "bf16":
        monkeypatch.setattr(four, "gemm_impl", "bf16")
    else:
        monkeypatch.setattr(four, "mx4_activations", kind)
    k, n = 640, 333
    lin = four.Linear(k, n, bias=True).cuda()
    w = _fill(lin, g)["weight"]
    x = torch.randn(2, m, k, generator=g).bfloat16().cuda()
    with torch.no_grad():
        y = lin(x)
        bias = lin.bias.data
        if kind == "bf16":
            assert torch.equal(y, F.linear(x, w, bias))
            return
        a, a_s = kernel.act_quant(x, 128, "ue8m0") if kind == "e4m3" else kernel.mx4_quant(x)
        assert torch.equal(y, kernel.mx4_gemm(a, a_s, lin.weight, lin.scale) + bias)
    ref = x.double() @ w.double().t() + bias.double()
    if kind == "e4m3":
        top = x.abs().double().unflatten(-1, (-1, 128)).amax(-1, keepdim=True).expand(-1, -1, -1, 128).flatten(-2)
        off = torch.maximum(x.abs().double() * 2.0 ** -4, top * 2.0 ** -17)         # a scale is at most 2 / 448 of the largest, half a step of 2^-9
    else:
        scale = a_s.float().double().repeat_interleave(32, -1)
        off = torch.maximum(x.abs().double(), scale) / 4
    bound = off @ w.abs().double().t() + 2.0 ** -7 * (ref.abs() + bias.abs().double() + off @ w.abs().double().t()) + 2.0 ** -10 * (x.abs().double() @ w.abs().double().t())
    assert ((y.double() - ref).abs() <= bound).all()


def test_feed_forward_block(four):
    """Its three linear layers and the two operations between them, one after the other."""
    g = torch.Generator().manual_seed(5)
    mlp = four.MLP(256, 384).cuda()
    _fill(mlp, g)
    x = torch.randn(9, 256, generator=g).bfloat16().cuda()
    with torch.no_grad():
        y = mlp(x)
        lin = four.linear
        w1, w2, w3 = (m.weight for m in (mlp.w1, mlp.w2, mlp.w3))
        assert torch.equal(y, lin(F.silu(lin(x, w1)) * lin(x, w3), w2)) and y.abs().max() > 0
        # one layer of 8 bits among them: still every layer on its own
        mlp.w2 = four.RowParallelLinear(384, 256, dtype=FP8).cuda()
        from dsv3fp8 import weight_quant
        mlp.w2.weight.data, mlp.w2.scale.data = weight_quant(torch.randn(256, 384, generator=g).bfloat16().cuda())
        assert torch.equal(mlp(x), lin(F.silu(lin(x, w1)) * lin(x, w3), mlp.w2.weight))


def test_experts(four):
    """Experts of 4-bit weights, routed to one by one."""
    g = torch.Generator().manual_seed(6)
    args = four.ModelArgs(dim=256, moe_inter_dim=128, n_routed_experts=4, n_activated_experts=2, n_expert_groups=1, n_limited_groups=1)
    moe = four.MoE(args).cuda()
    _fill(moe, g)
    x = torch.randn(2, 5, 256, generator=g).bfloat16().cuda()
    with torch.no_grad():
        y = moe(x)
        flat = x.view(-1, 256)
        weights, indices = moe.gate(flat)
        want = torch.zeros_like(flat)
        for i in range(4):
            at, top = torch.where(indices == i)
            if at.numel():
                want[at] += moe.experts[i](flat[at]) * weights[at, top, None]
        assert torch.equal(y.view(-1, 256), want + moe.shared_experts(flat))


@pytest.mark.parametrize("rank", [128, 0])
def test_attention_layer(four, monkeypatch, rank):
    """A layer of 4-bit weights and the same layer of the bf16 weights that they stand for: inputs of its linear layers are e4m3 in the one."""
    g = torch.Generator().manual_seed(7)
    args = four.ModelArgs(dim=256, n_heads=4, q_lora_rank=rank, max_batch_size=2, max_seq_len=32)
    layer = four.MLA(args).cuda()
    values = _fill(layer, g)
    monkeypatch.setattr(four.Linear, "dtype", torch.bfloat16)
    wide = four.MLA(args).cuda()
    for name, p in wide.named_parameters():
        p.data.copy_(values[name] if name in values else dict(layer.named_parameters())[name].data)
    x, freqs = torch.randn(2, 6, 256, generator=g).bfloat16().cuda(), _freqs(ROPE, 32).cuda()
    mask = torch.full((6, 6), float("-inf"), device="cuda").triu_(1)
    with torch.no_grad():
        y, ref = layer(x, 0, freqs[:6], mask).double(), wide(x, 0, freqs[:6], mask).double()
    # three linear layers behind each other, e4m3 inputs (2^-4 at most, 2^-5 on average, which random products keep), and the scores, which are small
    assert ((y - ref).norm(dim=-1) <= 3 * 2.0 ** -4 * ref.norm(dim=-1)).all() and ref.norm() > 0


def _pages(monkeypatch):
    """The tests of the layer on pages take their caches from here."""
    from dsv3fp8 import model
    plain = model.LatentPages
    monkeypatch.setattr(model, "LatentPages", lambda *a, **k: plain(*a, **k, bits=4))


def test_prompt_tokens_tree_and_accepted_path(M, monkeypatch):  # noqa: F811
    _pages(monkeypatch)
    eight.test_prompt_tokens_tree_and_accepted_path(M)


@pytest.mark.parametrize("s", [1, 30, 64, 65, 130])
def test_prompts_and_the_token_behind_them(M, s):  # noqa: F811
    """Two sequences, one of half the length, in pages that end inside a tile; then a token each."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 51), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(s)
    cache = LatentPages(20, 24, device="cuda", bits=4)
    table = torch.randperm(20, generator=g)[:14].view(2, 7).int().cuda()
    lengths = [0, 0]
    for n, counts in ((s, (s, (s + 1) // 2)), (1, (1, 1))):
        starts, count = _ints(*lengths), _ints(*counts)
        x, freqs = _tokens(g, 2, n, [[k + t for t in range(n)] for k in lengths])
        positions = max(lengths) + n
        ref = _reference(layer, x, cache, table, starts, count, freqs, positions, lambda i, t: range(t + 1))
        with torch.inference_mode():
            y = layer.forward_paged(x, cache, table, starts, count, freqs, positions)
        _check(y, ref, count)
        lengths = [k + c for k, c in zip(lengths, counts)]


@pytest.mark.parametrize("s", [3, 70])
def test_rows_that_are_not_finite_reach_the_tokens_that_see_them(M, s):  # noqa: F811
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 53), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(54)
    table = torch.tensor([[3, 1, 5, 0], [2, 4, 6, 7]], dtype=torch.int32).cuda()
    x, freqs = _tokens(g, 2, s, [list(range(s))] * 2)
    out = []
    for bad in (False, True):
        cache = LatentPages(8, 24, device="cuda", bits=4)
        if bad:
            x[0, 1] = float("nan")              # its query and its row
        with torch.inference_mode():
            out.append(layer.forward_paged(x, cache, table, _ints(0, 0), _ints(s, s), freqs, s))
    clean, got = out
    assert torch.equal(got[0, 0], clean[0, 0]) and got[0, 1:].isnan().all() and torch.equal(got[1], clean[1])


def test_a_captured_step_serves_every_length(M):  # noqa: F811
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 45), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(46)
    cache, other = LatentPages(8, 16, device="cuda", bits=4), LatentPages(8, 16, device="cuda", bits=4)
    table = torch.tensor([[2, 7, 1], [0, 4, 5]], dtype=torch.int32).cuda()
    x, freqs = _tokens(g, 2, 1, [[0], [0]])
    starts, counts = _ints(0, 0), _ints(1, 1)
    raw = lambda c: (c.kv.view(torch.uint8), c.scale.view(torch.uint8), c.pe)  # noqa: E731
    with torch.inference_mode():
        layer.forward_paged(x, other, table, starts, counts, freqs, 48)
        for mine, warm in zip(raw(cache), raw(other)):
            mine.copy_(warm)
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
    for a, c in zip(raw(cache), raw(other)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("s,what", [(3, "block"), (3, "first block"), (3, "last block"), (70, "block"), (70, "first block"), (70, "last block"), (70, "infinity")])
def test_rows_of_which_a_part_is_not_finite_reach_the_tokens_that_see_them(M, s, what):  # noqa: F811
    """A cached row from elsewhere with one scale of NaN, or (in a prompt, which reads rows as bf16) with a number of 2^128: NaN for the tokens of its sequence, which all see
    it, and the bits that they get without it for the others'."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 55), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(56)
    table = torch.tensor([[3, 1, 5, 0, 9], [2, 4, 6, 7, 8]], dtype=torch.int32).cuda()
    first, freqs0 = _tokens(g, 2, 40, [list(range(40))] * 2)
    x, freqs = _tokens(g, 2, s, [list(range(40, 40 + s))] * 2)
    out = []
    for bad in (False, True):
        cache = LatentPages(10, 24, device="cuda", bits=4)
        with torch.inference_mode():
            layer.forward_paged(first, cache, table, _ints(0, 0), _ints(40, 40), freqs0, 40)
            if bad:
                row = cache.scale.view(torch.uint8)[1, 9], cache.kv.view(torch.uint8)[1, 9]           # position 33 of sequence 0
                if what == "infinity":
                    row[0].fill_(245)
                    row[0][11], row[1][11 * 16 + 5] = 253, 0x60                                          # 4 * 2^126
                else:
                    row[0][{"block": 9, "first block": 0, "last block": 15}[what]] = 255
            out.append(layer.forward_paged(x, cache, table, _ints(40, 40), _ints(s, s), freqs, 40 + s))
    clean, got = out
    assert clean.isfinite().all() and got[0].isnan().all() and torch.equal(got[1].view(torch.int16), clean[1].view(torch.int16))


def test_a_prompt_captured_and_replayed(M):  # noqa: F811
    """One graph of a prompt's step on 4-bit rows; rows of which a block is NaN come and go between the replays."""
    from dsv3fp8.model import LatentPages
    layer = _layer(M, small_mla_params(DIM, HEADS, RANK, C, NOPE, ROPE, V, 57), DIM, HEADS, RANK, 8)
    g = torch.Generator().manual_seed(58)
    table = torch.tensor([[3, 1, 5, 0, 9], [2, 4, 6, 7, 8]], dtype=torch.int32).cuda()
    cache, start, other = (LatentPages(10, 24, device="cuda", bits=4) for _ in range(3))
    raw = lambda c: (c.kv.view(torch.uint8), c.scale.view(torch.uint8), c.pe)  # noqa: E731
    first, freqs0 = _tokens(g, 2, 40, [list(range(40))] * 2)
    x, freqs = _tokens(g, 2, 70, [list(range(40, 110))] * 2)
    starts, counts = _ints(40, 40), _ints(70, 70)
    with torch.inference_mode():
        layer.forward_paged(first, start, table, _ints(0, 0), _ints(40, 40), freqs0, 40)
        layer.forward_paged(x, other, table, starts, counts, freqs, 120)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward_paged(x, cache, table, starts, counts, freqs, 120)
        for step in range(6):
            x.copy_(_tokens(g, 2, 70, [list(range(70))] * 2)[0])
            for c in (cache, other):
                for mine, theirs in zip(raw(c), raw(start)):
                    mine.copy_(theirs)
                if step % 2:
                    raw(c)[1][4, 3, step] = 255                     # position 27 of sequence 1
            graph.replay()
            want = layer.forward_paged(x, other, table, starts, counts, freqs, 120)
            torch.cuda.synchronize()
            assert torch.equal(y.view(torch.int16), want.view(torch.int16))
            assert y[0].isfinite().all() and (y[1].isnan().all() if step % 2 else y[1].isfinite().all())


def test_conversions_of_a_layer_leave_its_codes(four):
    """Moved and converted as a whole, with another layer and a bias: the same products."""
    g = torch.Generator().manual_seed(8)
    lin = four.Linear(256, 48, bias=True)
    block = torch.nn.Sequential(lin, torch.nn.LayerNorm(48)).cuda()
    _fill(lin, g)
    codes, scale = lin.weight.data.view(torch.uint8).clone(), lin.scale.data.view(torch.uint8).clone()
    x = torch.randn(5, 256, generator=g).bfloat16().cuda()
    with torch.no_grad():
        want = lin(x)
        block.float()
        assert lin.bias.dtype == torch.float32
        block.to("cpu", torch.float16).to("cuda", torch.bfloat16)
        assert lin.weight.is_cuda and lin.scale.is_cuda and lin.weight.scale is lin.scale and lin.bias.dtype == torch.bfloat16
        assert torch.equal(lin.weight.data.view(torch.uint8), codes) and torch.equal(lin.scale.data.view(torch.uint8), scale)
        assert torch.equal(lin(x), want)
