"""The latent cache in pages of 4-bit rows on the GPU: rows written, read back, moved and attended to, against plain evaluations on the host and against the
attention on e4m3 rows of the same values, which are its own operands."""
import pytest
import torch

from test_gpu_mla_paged import (ATTEND, C, EPS, NOPE, READ, ROPE, V, WRITE, _attention_case, _attention_reference, _bits, _close, _phases, _rotated, _rows,
                                _tables)
from test_gpu_mx4 import VALUES, held, packed, quantised

pytestmark = pytest.mark.gpu

FP8, FP4, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


@pytest.fixture(scope="module", autouse=True)
def _ops():
    from dsv3fp8 import ops  # noqa: F401  (registers torch.ops.dsv3fp8)


def _row_codes(x):
    """Packed codes and scale bytes of cache rows: none of a row's scales more than 14 powers of two below its largest, all NaN where one is."""
    _, byte = quantised(x)
    byte = byte.int()
    top = byte.amax(-1, keepdim=True)
    byte = torch.where(top == 255, 255, torch.maximum(byte, top - 14))
    v = x.double().nan_to_num(0.0, 0.0, 0.0).unflatten(-1, (-1, 32)) * torch.exp2(127.0 - byte.double())[..., None]
    gap = (v.abs()[..., None] - VALUES[:8]).abs()
    code = (gap + torch.tensor([0.0, 1e-12] * 4, dtype=torch.float64)).argmin(-1) | torch.where(torch.signbit(v), 8, 0)
    return packed(torch.where(byte[..., None] == 255, 0, code).flatten(-2)), byte.to(torch.uint8)


def _pool(g, pages, page, spread=6):
    """A cache whose rows all hold something: random codes, scales up to `spread` powers of two below the row's largest, that one any."""
    n = pages * page
    codes = torch.randint(0, 256, (n, C // 2), generator=g).to(torch.uint8)
    top = torch.randint(118, 124, (n, 1), generator=g)
    scale = top - torch.randint(0, spread + 1, (n, C // 32), generator=g)
    return [codes.view(pages, page, C // 2).view(FP4), scale.to(torch.uint8).view(pages, page, C // 32).view(E8M0),
            torch.randn(pages, page, ROPE, generator=g).bfloat16()]


def _write_reference(a, qn, kn, freqs, kv, scale, pe, table, starts, counts):
    def norm(x, w):
        r = (1 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
        return (x.float() * r * w.float()).bfloat16().float()
    qr = 0 if qn is None else qn.numel()
    kv, scale, pe = kv.clone(), scale.clone(), pe.clone()
    pages, page = kv.shape[:2]
    codes, s = _row_codes(norm(a[..., qr:qr + C], kn))
    key = _rotated(a[..., qr + C:], freqs).bfloat16()
    for b in range(a.size(0)):
        if starts[b] < 0:
            continue
        for i, row in enumerate(_rows(table, page, pages, b, range(int(starts[b]), int(starts[b]) + min(int(counts[b]), a.size(1))))):
            if row >= 0:
                kv.view(torch.uint8).view(-1, C // 2)[row] = codes[b, i]
                scale.view(torch.uint8).view(-1, C // 32)[row] = s[b, i]
                pe.view(-1, ROPE)[row] = key[b, i]
    if qr:
        n = norm(a[..., :qr], qn).unflatten(-1, (-1, 128))
        ys = n.abs().amax(-1).clamp_min(1e-4) / torch.tensor(448.0)
        return kv, scale, pe, (n / ys[..., None]).to(FP8).flatten(-2), ys
    return kv, scale, pe, a.new_empty(*a.shape[:2], 0, dtype=FP8), a.new_empty(*a.shape[:2], 0, dtype=torch.float32)


@pytest.mark.parametrize("b,s,qr,page", WRITE)
def test_rows_are_quantised_as_they_are_written(b, s, qr, page):
    g = torch.Generator().manual_seed(b * 100 + s)
    starts = torch.randint(0, 90, (b,), generator=g).int()
    counts = torch.randint(0, s + 1, (b,), generator=g).int()
    starts[0], counts[0] = 37, s
    if b > 3:
        counts[1], counts[2], starts[3] = -5, s + 9, -2              # nothing, all rows, nothing
    lengths = [max(0, int(x)) + s for x in starts]
    pages = sum(-(-n // page) for n in lengths) + 1
    table = _tables(g, lengths, page, pages)
    if b > 1:
        table[1, 0] = pages                                          # no page: its rows are left out
    a = torch.randn(b, s, qr + C + ROPE, generator=g).bfloat16() * 3
    a[0, 0, qr:qr + C] = 0                                            # a row of zeros
    if s > 2:
        a[0, 1, qr + 3], a[0, 2, qr + 77] = float("nan"), float("inf")
    if s > 4:
        a[0, 3, qr + 32:qr + C] *= 2.0 ** -18                         # blocks far below the row's largest
        a[0, 4, qr + 64:qr + 96] *= 2.0 ** -15
    qn = (1 + 0.1 * torch.randn(qr, generator=g)).bfloat16() if qr else None
    kn = (1 + 0.1 * torch.randn(C, generator=g)).bfloat16()
    pool = _pool(g, pages, page)
    freqs = _phases(g, b, s)
    want = _write_reference(a, qn, kn, freqs, *pool, table, starts, counts)
    dev = [t.cuda() for t in pool]
    y, ys = torch.ops.dsv3fp8.mla_latent_paged(a.cuda(), None if qn is None else qn.cuda(), kn.cuda(), freqs.cuda(), *dev, table.cuda(), starts.cuda(), counts.cuda(), EPS, EPS)
    # the same roundings in the same places, the root's sum in binary64: bit for bit
    for got, ref in zip((*dev, y, ys), want):
        same = _bits(got) == _bits(ref)
        if got.dtype in (torch.bfloat16, torch.float32):
            same |= torch.isnan(got.float().cpu()) & torch.isnan(ref.float())
        assert same.all()
    if s > 2:
        bad = _rows(table, page, pages, 0, [38, 39])
        assert (_bits(dev[1]).view(-1, 16)[bad] == 255).all() and (_bits(dev[0]).view(-1, C // 2)[bad] == 0).all()


@pytest.mark.parametrize("lengths,positions,page", READ)
def test_rows_are_read_back(lengths, positions, page):
    g = torch.Generator().manual_seed(positions)
    b, n = len(lengths), [max(0, x) for x in lengths]
    pages = sum(-(-x // page) for x in n) + 1
    table, pool = _tables(g, n, page, pages), _pool(g, pages, page, 14)
    if n[-1] > page:
        table[-1, 1] = -1                                            # a page that the sequence does not have
    pool[1].view(torch.uint8)[0, 0] = 255                            # a row that was not finite
    kv, pe = torch.ops.dsv3fp8.mla_cache_read(*[t.cuda() for t in pool], table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), positions)
    assert kv.shape == (b, positions, C) and pe.shape == (b, positions, ROPE)
    want_kv, want_pe = torch.zeros(b, positions, C), torch.zeros(b, positions, ROPE).bfloat16()
    values = held(*pool[:2]).view(-1, C)
    for i in range(b):
        row = _rows(table, page, pages, i, range(min(n[i], positions)))
        live = (row >= 0).nonzero().flatten()
        want_kv[i, live] = values[row[live]].float()
        want_pe[i, live] = pool[2].view(-1, ROPE)[row[live]]
    want = want_kv.bfloat16()
    assert torch.equal(want.isnan(), kv.cpu().isnan())
    assert torch.equal(want.nan_to_num(7.0), kv.cpu().nan_to_num(7.0)) and torch.equal(_bits(pe), _bits(want_pe))


@pytest.mark.parametrize("page", [8, 24])
@pytest.mark.parametrize("b,most", [(1, 1), (3, 9), (70, 3), (2, 64)])
def test_accepted_rows_are_moved(b, most, page):
    g = torch.Generator().manual_seed(b + most + page)
    starts = torch.randint(0, 50, (b,), generator=g).int()
    path = torch.stack([torch.randperm(64, generator=g)[:most] for _ in range(b)]).int()       # in any order, one over the other
    kept = torch.randint(0, most + 1, (b,), generator=g).int()
    kept[0] = most
    if b > 2:
        kept[1], starts[2] = most + 7, -1
        path[0, 1], path[0, 2] = path[0, 0], -4                      # one row twice; none
    lengths = [max(0, int(x)) + 64 for x in starts]
    pages = sum(-(-n // page) for n in lengths) + 1
    table, pool = _tables(g, lengths, page, pages), _pool(g, pages, page)
    if b > 2:
        table[1, 0] = -1
    want = [t.clone() for t in pool]
    for i in range(b):
        if starts[i] < 0:
            continue
        for k in range(min(int(kept[i]), most)):
            if path[i, k] < 0:
                continue
            src, dst = _rows(table, page, pages, i, [int(starts[i] + path[i, k]), int(starts[i] + k)]).tolist()
            if src >= 0 and dst >= 0:
                for t, w in zip(pool, want):
                    w.view(torch.uint8).view(pages * page, -1)[dst] = t.view(torch.uint8).view(pages * page, -1)[src]
    dev = [t.cuda() for t in pool]
    torch.ops.dsv3fp8.mla_cache_keep(*dev, table.cuda(), starts.cuda(), path.cuda(), kept.cuda())
    for got, ref in zip(dev, want):
        assert torch.equal(_bits(got), _bits(ref))


# ------------------------------------------------------------------------------------------------------------ attention

def _as_e4m3(kv, scale):
    """The same rows as e4m3 codes of one scale: 2^6 times the code where the block has the row's largest scale, 2^-8 times it 14 powers below."""
    byte = scale.view(torch.uint8).int()
    top = byte.amax(-1, keepdim=True)
    one = kv.view(torch.uint8).long()
    v = VALUES[torch.stack((one & 15, one >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32)) * torch.exp2((6 + byte - top).double())[..., None]
    codes = v.flatten(-2).float().to(FP8)
    assert torch.equal(codes.double(), v.flatten(-2))
    return codes, torch.where(top == 255, float("nan"), torch.exp2((top - 133).double())).squeeze(-1).float()


def _case(b, s, h, context, page, kind, seed, spread=6):
    """A case of the attention on e4m3 rows with a pool of 4-bit ones: their arguments, those of the same rows in e4m3, what is seen.  Rows that nobody sees hold NaN."""
    args, seen = _attention_case(b, s, h, context, page, kind, seed)
    g = torch.Generator().manual_seed(seed + 1)
    pages = args[3].size(0)
    kv, scale, _ = _pool(g, pages, page, spread)
    lost = (args[2].cpu().view(torch.uint8) == 0x7f).all(-1)
    scale.view(torch.uint8)[lost] = 255
    kv.view(torch.uint8)[lost] = 0
    e4m3, row_scale = _as_e4m3(kv, scale)
    rest = args[4:]
    return [*args[:2], kv.cuda(), scale.cuda(), *rest], [*args[:2], e4m3.cuda(), row_scale.cuda(), *rest], seen


@pytest.mark.parametrize("b,s,h,context,page,kind", ATTEND)
def test_attention(b, s, h, context, page, kind):
    """Bit for bit what the attention on e4m3 rows gives for the same values, and close to an evaluation in 64 bits."""
    four, eight, seen = _case(b, s, h, context, page, kind, b + s + context, 14 if s == 1 else 5)
    got = torch.ops.dsv3fp8.mla_decode_paged(*four)
    assert torch.isfinite(got).all()
    assert torch.equal(_bits(got), _bits(torch.ops.dsv3fp8.mla_decode_paged(*eight)))
    assert _close(got.view(b, s, h, V).double(), _attention_reference([*eight[:3], eight[3].nan_to_num(1.0), *eight[4:]], seen))


@pytest.mark.parametrize("b,s,h,context,page,kind", [(1, 1, 128, 33, 64, None), (3, 13, 24, 200, 24, "any"), (2, 9, 128, 200, 40, "tree")])
def test_attention_quantised_is_the_rounded_result_quantised(b, s, h, context, page, kind):
    from dsv3fp8 import kernel
    four, _, _ = _case(b, s, h, context, page, kind, 5)
    y = torch.ops.dsv3fp8.mla_decode_paged(*four)
    yq, ys = torch.ops.dsv3fp8.mla_decode_paged_quant(*four)
    rq, rs = kernel.act_quant(y)
    assert torch.equal(yq.view(torch.uint8), rq.view(torch.uint8)) and torch.equal(ys.view(torch.int32), rs.view(torch.int32))


@pytest.mark.parametrize("h,page", [(128, 64), (6, 24), (2, 40)])
def test_rows_that_are_not_finite_reach_those_who_see_them(h, page):
    four, _, seen = _case(2, 12, h, 150, page, "tree", 11)
    clean = torch.ops.dsv3fp8.mla_decode_paged(*four)
    first, pages = int(four[6][0]), four[3].size(0)
    row = lambda j: int(_rows(four[5].cpu(), page, pages, 0, [j])[0])  # noqa: E731
    for what in ("latent", "block", "nan key"):
        node = 7
        kv, scale, pe = four[2].clone(), four[3].clone(), four[4].clone()
        if what == "latent":
            kv.view(torch.uint8).view(-1, C // 2)[row(first + node)] = 0
            scale.view(torch.uint8).view(-1, 16)[row(first + node)] = 255
        elif what == "block":
            scale.view(torch.uint8).view(-1, 16)[row(first + node), 9] = 255
        else:
            pe.view(-1, ROPE)[row(first + node), 3] = float("nan")
        got = torch.ops.dsv3fp8.mla_decode_paged(four[0], four[1], kv, scale, pe, *four[5:])
        for t in range(12):
            if node in seen[0][t]:
                assert torch.isnan(got[0, t]).all()
            else:
                assert torch.equal(_bits(got[0, t]), _bits(clean[0, t]))
        assert torch.equal(_bits(got[1]), _bits(clean[1]))


@pytest.mark.parametrize("h", [20, 8])
@pytest.mark.parametrize("page", [8, 40, 64])
def test_attention_skips_what_is_no_page(page, h):
    four, eight, seen = _case(3, 4, h, 230, page, "tree", 2)
    pages = four[3].size(0)
    for i, k, entry in ((0, 1, -1), (0, 2, pages), (2, 0, 2 ** 31 - 1), (1, 0, -7)):
        if k < four[5].size(1):
            four[5][i, k] = entry
    got = torch.ops.dsv3fp8.mla_decode_paged(*four)
    assert torch.equal(_bits(got), _bits(torch.ops.dsv3fp8.mla_decode_paged(*eight)))       # (the table is theirs too)
    assert _close(got.view(3, 4, h, V).double(), _attention_reference([*eight[:3], eight[3].nan_to_num(1.0), *eight[4:]], seen))


@pytest.mark.parametrize("h", [64, 8])
def test_rows_of_the_smallest_and_largest_scales(h):
    """Rows whose largest scale is one of the least there are: zeros, and what binary32 has of numbers of 2^-127; rows of large ones."""
    four, _, _ = _case(2, 2, h, 200, 24, None, 3)
    scale = four[3].view(torch.uint8)
    for lo, hi in ((0, 3), (5, 9), (100, 101)):
        scale.copy_(torch.randint(lo, hi, scale.shape).to(torch.uint8))
        four[0][:] = torch.randn_like(four[0].float()).bfloat16()
        four[4].nan_to_num_(0.0)
        got = torch.ops.dsv3fp8.mla_decode_paged(*four)
        e4m3, row_scale = _as_e4m3(four[2].cpu(), four[3].cpu())
        if lo == 100:
            eight = [*four[:2], e4m3.cuda(), row_scale.cuda(), *four[4:]]
            assert torch.equal(_bits(got), _bits(torch.ops.dsv3fp8.mla_decode_paged(*eight)))
        else:
            assert (got.abs() < 1e-30).all()


@pytest.mark.parametrize("s,h", [(1, 20), (2, 6), (3, 128)])
def test_rows_whose_scales_lie_far_apart(s, h):
    """Rows from elsewhere, up to 60 powers of two between a row's scales: read back as they are; attended to as the e4m3 numbers, of 2^6 for the largest scale,
    that are nearest to them."""
    four, eight, _ = _case(2, s, h, 200, 24, None, 31)
    four[4].nan_to_num_(0.0)
    scale = torch.randint(60, 121, four[3].shape, generator=torch.Generator().manual_seed(s)).to(torch.uint8)
    scale[..., 3:9] = torch.randint(100, 121, scale[..., 3:9].shape, generator=torch.Generator().manual_seed(h)).to(torch.uint8)
    four[3] = scale.cuda().view(E8M0)
    top = scale.int().amax(-1)
    value = held(four[2].cpu(), four[3].cpu())
    codes = (value * torch.exp2((133 - top).double())[..., None]).float().to(FP8)
    same = [*four[:2], codes.cuda(), torch.exp2((top - 133).double()).float().cuda(), *four[4:]]
    assert torch.equal(_bits(torch.ops.dsv3fp8.mla_decode_paged(*four)), _bits(torch.ops.dsv3fp8.mla_decode_paged(*same)))
    kv, _ = torch.ops.dsv3fp8.mla_cache_read(*four[2:5], torch.arange(four[2].size(0), dtype=torch.int32).cuda()[:, None], torch.full((four[2].size(0),), 24, dtype=torch.int32).cuda(), 24)
    assert torch.equal(kv.cpu(), value.bfloat16())


def test_attention_past_the_stated_positions_and_negative_starts():
    four, eight, _ = _case(4, 3, 16, 200, 16, None, 4)
    for args in (four, eight):
        args[11] = 150                                              # the longest sequence is cut there
    four[6][2] = -5                                                 # nothing
    got = torch.ops.dsv3fp8.mla_decode_paged(*four)
    assert (got[2] == 0).all() and torch.equal(_bits(got), _bits(torch.ops.dsv3fp8.mla_decode_paged(*eight)))


@pytest.mark.parametrize("h", [16, 8])
def test_attention_past_32_bits_of_bytes(h):
    """A pool of more than 2^32 bytes of codes, pages from its end: written, read, attended to."""
    page, pages = 8192, 2100
    kv = torch.zeros(pages, page, C // 2, dtype=torch.uint8, device="cuda")
    scale = torch.full((pages, page, 16), 127, dtype=torch.uint8, device="cuda")
    pe = torch.zeros(pages, page, ROPE, dtype=torch.bfloat16, device="cuda")
    assert kv.numel() > 2 ** 32
    g = torch.Generator().manual_seed(h)
    b, s, n = 2, 3, 9000
    kn = torch.ones(C).bfloat16().cuda()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows, freqs = torch.randn(b, n, C + ROPE, generator=g).bfloat16().cuda(), _phases(g, b, n).cuda()
    small = [torch.zeros(4, page, C // 2, dtype=torch.uint8, device="cuda").view(FP4), torch.full((4, page, 16), 127, dtype=torch.uint8, device="cuda").view(E8M0),
             torch.zeros(4, page, ROPE, dtype=torch.bfloat16, device="cuda")]
    large = [kv.view(FP4), scale.view(E8M0), pe]
    q = torch.randn(b, s, h, NOPE + ROPE, generator=g).bfloat16().cuda()
    w8, ws = torch.randn(h * (NOPE + V), C, generator=g).to(FP8).cuda(), (torch.rand(h * 2, C // 128, generator=g) * 0.03 + 0.01).cuda()
    out = []
    for pool, table in ((small, torch.tensor([[3, 0], [1, 2]])), (large, torch.tensor([[pages - 1, pages - 4], [pages - 3, pages - 2]]))):
        table = table.int().cuda()
        torch.ops.dsv3fp8.mla_latent_paged(rows, None, kn, freqs, *pool, table, i32(0, 0), i32(n, n - 700), EPS, EPS)
        back = torch.ops.dsv3fp8.mla_cache_read(*pool, table, i32(n, n - 700), n)
        y = torch.ops.dsv3fp8.mla_decode_paged(q, freqs[:, :s].contiguous(), *pool, table, i32(n - s, n - 700 - s), i32(s, s), None, w8, ws, n, 0.08)
        out.append((*back, y))
    for got, want in zip(*out):
        assert torch.equal(_bits(got), _bits(want))
    for k in range(3):
        assert torch.equal(_bits(large[k].view(torch.uint8)[pages - 4:].view(torch.uint8) if k < 2 else large[k][pages - 4:]), _bits(small[k].view(torch.uint8) if k < 2 else small[k]))


@pytest.mark.parametrize("b,s,h,context", [(3, 1, 128, 500), (2, 20, 16, 300), (3, 2, 16, 700)])
def test_a_step_captured_and_replayed(b, s, h, context):
    """Rows written, attended to, kept and read in one graph; two graphs; lengths, pages and queries change between replays."""
    cases = [_case(b, s, h, context, 24, "tree" if s > 1 else None, seed)[0] for seed in (1, 2, 3)]
    pages = max(c[3].size(0) for c in cases)

    def padded(c):
        c = list(c)
        for k in (2, 3, 4):
            t = c[k]
            raw = t.view(torch.uint8) if k < 4 else t
            big = torch.zeros(pages, *raw.shape[1:], dtype=raw.dtype, device="cuda")
            big[:t.size(0)] = raw
            c[k] = big.view(t.dtype)
        c[0] = c[0].nan_to_num(0.0)
        return c
    cases = [padded(c) for c in cases]
    g = torch.Generator().manual_seed(9)
    a = [torch.randn(b, s, C + ROPE, generator=g).bfloat16().cuda() for _ in cases]
    kn = torch.ones(C).bfloat16().cuda()
    path = torch.stack([torch.randperm(s, generator=g)[:min(4, s)] for _ in range(b)]).int().cuda()
    kept = torch.full((b,), min(3, s), dtype=torch.int32, device="cuda")

    def step(c, rows):
        torch.ops.dsv3fp8.mla_latent_paged(rows, None, kn, c[1], *c[2:8], EPS, EPS)
        y = torch.ops.dsv3fp8.mla_decode_paged(*c)
        torch.ops.dsv3fp8.mla_cache_keep(*c[2:7], path, kept)
        return y, *torch.ops.dsv3fp8.mla_cache_read(*c[2:6], c[6] + 1, context)

    def raw(t):
        return t.view(torch.uint8) if t.element_size() == 1 else t

    def fresh(c):
        return [raw(t).clone().view(t.dtype) if isinstance(t, torch.Tensor) else t for t in c]
    want = []
    for c, rows in zip(cases, a):
        c = fresh(c)
        want.append([raw(t).clone() for t in (*step(c, rows), *c[2:5])])
    graphs = []
    for _ in range(2):
        live, live_a = fresh(cases[0]), a[0].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(fresh(cases[0]), a[0])
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(live, live_a)
        graphs.append((graph, live, live_a, out))
    for k in (1, 2, 0, 1):
        for graph, live, live_a, out in graphs:
            for t, new in zip(live, cases[k]):
                if isinstance(t, torch.Tensor):
                    raw(t).copy_(raw(new))
            live_a.copy_(a[k])
            graph.replay()
            torch.ops.dsv3fp8.mla_decode_paged(*cases[k])           # eager work between the replays
        for _, live, _, out in graphs:
            for got, ref in zip((*out, *live[2:5]), want[k]):
                assert torch.equal(_bits(got), _bits(ref))


def test_two_streams_at_once():
    one, two = _case(8, 1, 128, 900, 64, None, 21)[0], _case(3, 20, 16, 400, 24, "tree", 22)[0]
    want = [torch.ops.dsv3fp8.mla_decode_paged(*a) for a in (one, two)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for k, a in enumerate((one, two)):
            with torch.cuda.stream(streams[k]):
                got[k].append(torch.ops.dsv3fp8.mla_decode_paged(*a))
    torch.cuda.synchronize()
    for k in (0, 1):
        for y in got[k]:
            assert torch.equal(_bits(y), _bits(want[k]))


@pytest.mark.parametrize("h", [64, 8])
@pytest.mark.parametrize("lo,hi,weights", [(0, 1, 100), (0, 3, 100), (5, 9, 100), (6, 20, 100), (100, 107, 0), (200, 206, -60), (225, 231, -80), (243, 247, -100), (240, 254, -100), (250, 254, -100), (253, 254, -100)])
def test_rows_of_scales_at_both_ends(lo, hi, weights, h):
    """Scales from 2^-127 to 2^126, the byte in front of the one that stands for no row, beside weights of 2^`weights` that bring the results to where bf16 has
    them: bit for bit the e4m3 rows of the same values, whose scale is 2^-6 times the row's largest (2^-125 the least), and as near to 64 bits as the scores' size lets them
    be.  Scores of the largest rows are so large that their rounding alone says which position is the largest; four and six times 2^126 are more than binary32 holds, in
    which the sums are: infinite there, or NaN."""
    four, _, seen = _case(2, 2, h, 200, 24, None, 3)
    g = torch.Generator().manual_seed(lo * 256 + hi)
    byte = torch.randint(lo, hi, four[3].shape, generator=g)
    byte[0, :, 0] = hi - 1
    four[0] = torch.randn(four[0].shape, generator=g).bfloat16().cuda()
    four[3] = byte.to(torch.uint8).cuda().view(E8M0)
    four[4].nan_to_num_(0.0)
    kv = four[2].view(torch.uint8)
    kv[:] = torch.randint(0, 256, kv.shape, generator=g).to(torch.uint8).cuda()
    four[10] = four[10] * 2.0 ** weights
    if lo >= 200:
        four[0][..., :NOPE] *= 2.0 ** (-(lo - 127) - weights if lo < 240 else -20)
    one = kv.cpu().long()
    values = VALUES[torch.stack((one & 15, one >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32))
    base = byte.amax(-1, keepdim=True).clamp_min(8)
    wide = (values * torch.exp2((6 + byte - base).double())[..., None]).flatten(-2)
    codes, row_scale = wide.float().to(FP8), torch.exp2((base - 133).double()).squeeze(-1).float()
    assert torch.equal(codes.double(), wide)
    eight = [*four[:2], codes.cuda(), row_scale.cuda(), *four[4:]]
    got = torch.ops.dsv3fp8.mla_decode_paged(*four)
    assert torch.equal(_bits(got), _bits(torch.ops.dsv3fp8.mla_decode_paged(*eight)))
    ref = _attention_reference(eight, seen)
    live = ref.abs().amax(-1) > 0
    got = got.view(ref.shape).double()
    assert live.any() and (got[~live] == 0).all()
    if hi <= 250:
        assert got.isfinite().all() and (got[live].abs().amax(-1) > 2.0 ** -60).all()
    if hi < 240:
        assert ((got - ref).norm(dim=-1) <= 2.0 ** -7 * ref.norm(dim=-1) + _at_both_ends(eight, seen)).all()


def _at_both_ends(args, seen):
    """What numbers near binary32's smallest and scores of any size add to an attention's error, as a norm [b, s, h].  Exponentials times their row's scale 2^r are pairs of e4m3 codes whose second
    one has a scale of 2^-126 at least: off by half of 2^-9 of that, 2^-136, which is 2^(-136 - r) of an exponential.  The largest of these is above 1/2 (offsets
    are scores rounded up to whole numbers), so that a weight is off by 2^(-136 - r) * 2 * the largest weight.  And the sums of latents go into the last product as two bf16
    numbers, multiples of 2^-133: off by 2^-134 for each of 512.  A folded query is a pair of codes, off by 2^-9 of itself or 2^-21 of the largest beside it, and of the
    products of eight features 7 * 2^-13 of their sizes are cut: a score is off by d = softmax_scale * (sum |q| |c| (2^-9 + 7 * 2^-13) + 2^-21 max |q| sum |c|), and a weight
    by a factor of e^(d + the largest d) at most."""
    q, freqs, kv, scale, pe, table, starts, counts, _, w8, ws, positions, softmax_scale = args
    b, s, h, _ = q.shape
    pages, page = scale.shape
    w = (w8.float() * ws.repeat_interleave(128, 0).repeat_interleave(128, 1)).bfloat16().double().view(h, NOPE + V, C)
    out = torch.zeros(b, s, h, dtype=torch.float64, device=q.device)
    for i in range(b):
        first = int(starts[i])
        for t in range(int(counts[i])):
            rows = _rows(table.cpu(), page, pages, i, list(range(first)) + [first + j for j in sorted(seen[i][t])]).cuda()
            r = scale.view(-1)[rows].double()
            c, k = kv.view(-1, C)[rows].double() * r[:, None], pe.view(-1, ROPE)[rows].double()
            turned = _rotated(q[i, t, :, NOPE:], freqs[i, t, None]).bfloat16().double()
            for a in range(h):
                folded = q[i, t, a, :NOPE].double() @ w[a, :NOPE]
                p = ((folded @ c.T + turned[a] @ k.T) * softmax_scale).softmax(-1)
                d = softmax_scale * ((2.0 ** -9 + 7 * 2.0 ** -13) * (folded.abs() @ c.abs().T) + 2.0 ** -21 * folded.abs().max() * c.abs().sum(-1))
                off = p * torch.expm1(d + d.max()) + (2.0 ** -135 / r) * p.max()
                out[i, t, a] = (off * (c @ w[a, NOPE:].T).norm(dim=-1)).sum() + 2.0 ** -134 * w[a, NOPE:].abs().sum(-1).norm()
    return out


@pytest.mark.parametrize("size", [-133, -126, -120, -60, 60, 120, 126])
def test_rows_of_any_size_are_written_and_read(size):
    """Norm weights of 2^size: latents from binary32's subnormal numbers up to its largest, bit for bit."""
    g = torch.Generator().manual_seed(size + 200)
    b, s, page, pages = 2, 9, 8, 6
    table = torch.randperm(pages, generator=g)[:4].view(2, 2).int()
    starts, counts = torch.tensor([3, 0], dtype=torch.int32), torch.tensor([9, 9], dtype=torch.int32)
    a = torch.randn(b, s, C + ROPE, generator=g).bfloat16()
    a[0, 2, :C - 40] *= 2.0 ** -7
    kn = (torch.randn(C, generator=g) * 2.0 ** size).bfloat16().clamp(torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max)
    pool, freqs = _pool(g, pages, page), _phases(g, b, s)
    want = _write_reference(a, None, kn, freqs, *pool, table, starts, counts)
    dev = [t.cuda() for t in pool]
    torch.ops.dsv3fp8.mla_latent_paged(a.cuda(), None, kn.cuda(), freqs.cuda(), *dev, table.cuda(), starts.cuda(), counts.cuda(), EPS, EPS)
    for got, ref in zip(dev, want):
        assert torch.equal(_bits(got), _bits(ref))
    kv, _ = torch.ops.dsv3fp8.mla_cache_read(*dev, table.cuda(), torch.tensor([12, 9], dtype=torch.int32).cuda(), 12)
    values = held(*want[:2]).view(-1, C)
    for i, n in ((0, 12), (1, 9)):
        back = values[_rows(table, page, pages, i, range(n))].float().bfloat16()
        assert torch.equal(kv[i, :n].cpu().isnan(), back.isnan()) and torch.equal(kv[i, :n].cpu().nan_to_num(7.0), back.nan_to_num(7.0))
