"""MLA.forward_paged and LatentPages on the host: what they refuse, and which operators a call consists of (no kernel runs)."""
import pytest
import torch

from test_mla_dispatch import FP8, _OnGpu, layer  # noqa: F401  (layer: a fixture)


@pytest.mark.parametrize("pages,page", [(0, 64), (-1, 64), (4, 0), (4, 7), (4, 12), (4, 16392), (4, -8)])
def test_pools_that_there_are_not(pages, page):
    from dsv3fp8.model import LatentPages
    with pytest.raises(ValueError):
        LatentPages(pages, page)


def test_pool():
    from dsv3fp8.model import LatentPages
    c = LatentPages(3, 24)
    assert c.kv.shape == (3, 24, 512) and c.kv.dtype == FP8 and c.scale.shape == (3, 24) and c.scale.dtype == torch.float32
    assert c.pe.shape == (3, 24, 64) and c.pe.dtype == torch.bfloat16
    assert (c.kv.float() == 0).all() and (c.scale == 1).all()


def _arguments(b, s):
    from dsv3fp8.model import LatentPages
    x = torch.zeros(b, s, 256, dtype=torch.bfloat16).as_subclass(_OnGpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return [x, LatentPages(4, 64), torch.zeros(b, 2, dtype=torch.int32), i32(*[0] * b), i32(*[s] * b), torch.ones(b, s, 32, dtype=torch.complex64), 128]


@pytest.fixture
def calls(layer, monkeypatch):  # noqa: F811
    """The operators in front of and behind the attention as stand-ins that note their arguments."""
    from dsv3fp8 import model
    monkeypatch.setattr(model, "gemm_impl", "fp8")
    layer.qk_nope_head_dim, layer.qk_rope_head_dim, layer.v_head_dim, layer.kv_lora_rank = 128, 64, 128, 512
    layer.qk_head_dim, out = 192, []

    def note(name, result):
        return lambda *a: (out.append((name, a)), result(*a))[1]
    ops = torch.ops.dsv3fp8
    monkeypatch.setattr(model, "linear", lambda x, *a: x)
    monkeypatch.setattr(model, "fp8_gemm", note("gemm", lambda a, s, w, ws: torch.zeros(*a.shape[:-1], w.size(0), dtype=torch.bfloat16)))
    pair = lambda a, n: (torch.zeros(*a.shape[:2], n, dtype=FP8), torch.zeros(*a.shape[:2], 1))  # noqa: E731
    monkeypatch.setattr(ops, "mla_latent_paged", note("latent", lambda a, *r: pair(a, 128)))
    monkeypatch.setattr(ops, "mla_decode_paged_quant", note("decode", lambda q, *r: pair(q, 256)))
    monkeypatch.setattr(ops, "mla_prefill", note("prefill", lambda q, *r: pair(q, 256)))
    monkeypatch.setattr(ops, "mla_cache_read", note("read", lambda kv, sc, pe, table, n, t: (torch.zeros(table.size(0), t, 512), torch.zeros(table.size(0), t, 64))))
    return out


@pytest.mark.parametrize("b,s", [(2, 1), (1, 64), (3, 65)])
def test_operators_of_a_call(layer, calls, b, s):  # noqa: F811
    args = _arguments(b, s)
    tree = torch.ones(b, s, dtype=torch.int64) if s <= 64 else None
    with torch.no_grad():
        y = layer.forward_paged(*args, tree)
    assert y.shape == (b, s, 256)
    assert [c[0] for c in calls] == (["latent", "gemm", "decode", "gemm"] if s <= 64 else ["latent", "gemm", "read"] + ["prefill"] * b + ["gemm"])
    latent = calls[0][1]
    assert latent[1] is layer.q_norm.weight and latent[2] is layer.kv_norm.weight and latent[4] is args[1].kv and latent[7] is args[2]
    if s <= 64:
        decode = calls[2][1]
        assert decode[2] is args[1].kv and decode[5] is args[2] and decode[8] is tree and decode[9] is layer.wkv_b.weight and decode[11] == 128


@pytest.mark.parametrize("what", ["grad", "dtype", "shape", "freqs", "freqs shape", "wo", "wo hook", "norm", "dims", "gemm", "empty", "tree"])
def test_calls_that_are_refused(layer, calls, monkeypatch, what):  # noqa: F811
    from dsv3fp8 import model
    args, tree = _arguments(2, 3), None
    if what == "dtype":
        args[0] = args[0].float()
    elif what == "shape":
        args[0] = args[0][0]
    elif what == "freqs":
        args[5] = args[5].to(torch.complex128)
    elif what == "freqs shape":
        args[5] = args[5][0]
    elif what == "wo":
        layer.wo = torch.nn.Linear(256, 256)
    elif what == "wo hook":
        layer.wo.register_forward_hook(lambda *a: None)
    elif what == "norm":
        layer.kv_norm.eps = None
    elif what == "dims":
        layer.v_head_dim = 64
    elif what == "gemm":
        monkeypatch.setattr(model, "gemm_impl", "bf16")
    elif what == "empty":
        args = _arguments(2, 0)
    elif what == "tree":
        args, tree = _arguments(2, 65), torch.ones(2, 65, dtype=torch.int64)
    with torch.set_grad_enabled(what == "grad"), pytest.raises((RuntimeError, ValueError)):
        layer.forward_paged(*args, tree)
    assert not calls


@pytest.mark.parametrize("s", [1, 3, 64, 65, 200])
@pytest.mark.parametrize("positions", [0, -1, 129, 1 << 23, 2 ** 40])
def test_positions_that_the_table_has_no_room_for(layer, calls, s, positions):  # noqa: F811
    """Two pages of 64 a sequence; refused before a row is written, whatever the number of tokens."""
    args = _arguments(2, s)
    args[6] = positions
    if positions >= 1 << 23:                                # a table that would have room: more than the kernels count to
        args[2] = torch.zeros(1, 1, dtype=torch.int32).expand(2, positions // 64 + 1)
    with torch.no_grad(), pytest.raises(ValueError, match="positions"):
        layer.forward_paged(*args)
    assert not calls


@pytest.mark.parametrize("s", [3, 65])
def test_tables_of_another_shape(layer, calls, s):  # noqa: F811
    args = _arguments(2, s)
    args[2] = args[2][0]
    with torch.no_grad(), pytest.raises(ValueError, match="page_table"):
        layer.forward_paged(*args)
    assert not calls


@pytest.mark.parametrize("tree", [torch.ones(2, 3), torch.ones(2, 3, dtype=torch.int32), torch.ones(3, dtype=torch.int64), torch.ones(2, 4, dtype=torch.int64),
                                  torch.ones(1, 3, dtype=torch.int64), torch.ones(3, 2, dtype=torch.int64).t(), torch.ones(2, 3, dtype=torch.int64, device="meta")])
def test_trees_that_are_refused_before_a_row_is_written(layer, calls, tree):  # noqa: F811
    with torch.no_grad(), pytest.raises(ValueError, match="tree"):
        layer.forward_paged(*_arguments(2, 3), tree)
    assert not calls


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-40, float("inf"), float("nan")])
def test_scales_that_are_refused_before_a_row_is_written(layer, calls, scale):  # noqa: F811
    layer.softmax_scale = scale
    with torch.no_grad(), pytest.raises(RuntimeError, match="forward_paged"):
        layer.forward_paged(*_arguments(2, 3))
    assert not calls


def _masks(calls):
    return [c[1][6] for c in calls if c[0] == "prefill"]


@pytest.mark.parametrize("page,positions", [(64, 300), (8, 300), (24, 290), (512, 100), (16, 320)])
def test_prompts_do_not_see_what_lies_in_no_page(layer, calls, page, positions):  # noqa: F811
    """Position 0 in no page has the lowest number: nothing beside any other, a row of zeros for who sees no other."""
    from dsv3fp8.model import LatentPages
    width = -(-positions // page) + 1
    args, pages = _arguments(3, 70), 2 * width
    args[1], args[6] = LatentPages(pages, page), positions
    table = torch.randint(0, pages, (3, width), generator=torch.Generator().manual_seed(page)).int()
    table[0, 0], table[1, width // 2], table[1, width - 2], table[2, 0] = pages, -1, 2 ** 31 - 1, -2 ** 31
    args[2], args[3] = table, torch.tensor([5, 0, positions - 70], dtype=torch.int32)
    with torch.no_grad():
        layer.forward_paged(*args)
    masks = _masks(calls)
    assert len(masks) == 3
    at = torch.arange(positions)
    for i, mask in enumerate(masks):
        entry = table[i].long()[at // page]
        want = torch.zeros(70, positions).masked_fill((entry < 0) | (entry >= pages), float("-inf"))
        if not 0 <= entry[0] < pages:
            want[:, 0] = torch.finfo(torch.bfloat16).min
        want[at > args[3][i] + torch.arange(70)[:, None]] = float("-inf")
        assert mask.dtype == torch.bfloat16 and mask.is_contiguous() and torch.equal(mask.float(), want)


def test_prompts_see_rows_that_are_not_finite_and_no_others_do(layer, calls, monkeypatch):  # noqa: F811
    """Such rows go into the attention as zeros, with NaN in the mask for those who see them."""
    args, s, positions = _arguments(2, 70), 70, 128
    args[3] = torch.tensor([50, 0], dtype=torch.int32)
    kv, pe = torch.randn(2, positions, 512).bfloat16(), torch.randn(2, positions, 64).bfloat16()
    kv[0, 7], kv[1, 40] = float("nan"), float("nan")
    pe[0, 60, 3], pe[1, 41, 5], pe[1, 69, 63], pe[1, 100] = float("nan"), float("inf"), float("-inf"), float("nan")
    pe[0, 1, 2], kv[0, 1:3, 0] = torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).max       # (whose sum would be none)
    read = kv.clone(), pe.clone()
    monkeypatch.setattr(torch.ops.dsv3fp8, "mla_cache_read", lambda *a: read)
    with torch.no_grad():
        layer.forward_paged(*args)
    masks = _masks(calls)
    given = [c[1] for c in calls if c[0] == "prefill"]
    at, token = torch.arange(positions), torch.arange(s)[:, None]
    for i, bad in enumerate(([7, 60], [40, 41, 69, 100])):
        want = torch.zeros(s, positions)
        want[:, bad] = float("nan")
        want[at > args[3][i] + token] = float("-inf")
        assert torch.equal(masks[i].isnan(), want.isnan()) and torch.equal(masks[i][~want.isnan()].float(), want[~want.isnan()].float())
        good = torch.ones(positions, dtype=torch.bool)
        good[bad] = False
        for got, clean in zip(given[i][2:4], (kv[i:i + 1], pe[i:i + 1])):
            assert got.isfinite().all() and torch.equal(got[:, good], clean[:, good])


@pytest.mark.parametrize("start,count", [(50, 2 ** 31 - 1), (2 ** 31 - 1, 70), (2 ** 31 - 60, 2 ** 31 - 1), (0, 71), (127, -2 ** 31), (-5, -2 ** 31)])
def test_prompts_with_starts_and_counts_out_of_range(layer, calls, start, count):  # noqa: F811
    """A count above the rows is all rows; positions behind the stated ones are none: what a token sees has been read, and nothing else is in its mask."""
    args = _arguments(1, 70)
    args[3][0], args[4][0] = start, count
    with torch.no_grad():
        y = layer.forward_paged(*args)
    lengths, mask = next(c[1][4] for c in calls if c[0] == "read"), _masks(calls)[0]
    token, at = torch.arange(70)[:, None], torch.arange(128)
    mine = torch.arange(70) < count
    sees = at <= start + token
    assert lengths.dtype == torch.int32 and torch.equal(mask == 0, sees) and y.shape == (1, 70, 256)
    assert (not mine.any() or start < 0 or int(lengths[0]) > int(sees[mine].nonzero()[:, 1].max()))


@pytest.mark.parametrize("bits", [8, 4])
def test_prompts_see_rows_of_which_a_part_is_not_finite(layer, calls, monkeypatch, bits):  # noqa: F811
    """A 4-bit row has 16 scales, of which one may be NaN, and numbers that bf16 does not hold: such a row is marked wherever that part lies.  (An e4m3 row has one scale.)"""
    from dsv3fp8.model import LatentPages
    args, s, positions = _arguments(1, 70), 70, 128
    args[1], args[3] = LatentPages(4, 64, bits=bits), torch.tensor([50], dtype=torch.int32)
    kv, pe = torch.randn(1, positions, 512).bfloat16(), torch.randn(1, positions, 64).bfloat16()
    kv[0, 3] = float("nan")
    kv[0, 4, 1:3] = torch.finfo(torch.bfloat16).max                 # (finite)
    bad = [3]
    if bits == 4:
        for row, block in ((7, 0), (20, 1), (33, 9), (77, 15)):
            kv[0, row, 32 * block:32 * block + 32] = float("nan")
        kv[0, 41, 500], kv[0, 100, 0], kv[0, 101, 40:42] = float("inf"), float("-inf"), torch.tensor([float("inf"), float("-inf")])
        bad += [7, 20, 33, 41, 77, 100, 101]
    read = kv.clone(), pe.clone()
    monkeypatch.setattr(torch.ops.dsv3fp8, "mla_cache_read", lambda *a: read)
    with torch.no_grad():
        layer.forward_paged(*args)
    mask, given = _masks(calls)[0], next(c[1] for c in calls if c[0] == "prefill")
    want = torch.zeros(s, positions)
    want[:, bad] = float("nan")
    want[torch.arange(positions) > 50 + torch.arange(s)[:, None]] = float("-inf")
    assert torch.equal(mask.isnan(), want.isnan()) and torch.equal(mask[~want.isnan()].float(), want[~want.isnan()].float())
    good = torch.ones(positions, dtype=torch.bool)
    good[bad] = False
    assert given[2].isfinite().all() and torch.equal(given[2][:, good], kv[:, good])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("name", ["wq_a", "wkv_a", "wq_b", "wkv_b", "wo"])
def test_layers_with_a_projection_of_4_bits_are_refused(layer, calls, name, bits):  # noqa: F811
    """Before a row is written, and by their reason."""
    from dsv3fp8.model import LatentPages
    lin, args = getattr(layer, name), _arguments(2, 3)
    args[1] = LatentPages(4, 64, bits=bits)
    with torch.no_grad():
        layer.forward_paged(*args)
        assert calls
        calls.clear()
        setattr(layer, name, type(lin)(lin.in_features, lin.out_features, dtype=torch.float4_e2m1fn_x2))
        with pytest.raises(RuntimeError, match="e4m3 weights .none of 4 bits"):
            layer.forward_paged(*args)
    assert not calls
