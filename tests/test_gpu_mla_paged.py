"""The latent cache in pages on the GPU: rows written, read back, moved and attended to, against plain evaluations on the host."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
C, ROPE, NOPE, V = 512, 64, 128, 128
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _ops():
    from dsv3fp8 import ops  # noqa: F401  (registers torch.ops.dsv3fp8)


def _bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).cpu()


def _quantised(x):
    """e4m3 codes and one power of two per row of fp32 rows; a row that is not finite: zeros and NaN."""
    fine = x.isfinite().all(-1)
    s = (x.abs().amax(-1).clamp_min(1e-4) / torch.tensor(448.0)).double()
    s = torch.where(fine, torch.exp2(torch.frexp(s)[1] - (torch.frexp(s)[0] == 0.5).int()), float("nan"))
    codes = torch.where(fine[..., None], x.double() / s[..., None], 0.0).float().to(FP8)
    return codes, s.float()


def _phases(g, *shape):
    a = torch.rand(*shape, ROPE // 2, generator=g) * 6.28
    return torch.polar(torch.ones_like(a), a)


def _rotated(x, freqs):
    re, im = x.float().unflatten(-1, (-1, 2)).unbind(-1)
    return torch.stack((re * freqs.real - im * freqs.imag, re * freqs.imag + im * freqs.real), -1).flatten(-2)


def _pool(g, pages, page):
    """A cache whose rows all hold something."""
    kv, s = _quantised(torch.randn(pages * page, C, generator=g).bfloat16().float())
    return [kv.view(pages, page, C), s.view(pages, page), torch.randn(pages, page, ROPE, generator=g).bfloat16()]


def _tables(g, lengths, page, pages):
    """Pages in no order; -1 and other numbers that name none behind the last."""
    width = max(-(-n // page) for n in lengths) + 2
    order, at = torch.randperm(pages, generator=g).int(), 0
    table = torch.tensor([[-1, pages, 2 ** 31 - 1, -2 ** 31][k % 4] for k in range(width)], dtype=torch.int32).repeat(len(lengths), 1)
    for b, n in enumerate(lengths):
        k = -(-n // page)
        table[b, :k] = order[at:at + k]
        at += k
    assert at <= pages
    return table


def _rows(table, page, pages, b, positions):
    """Cache rows of a sequence's positions, -1 where there is none."""
    out = []
    for j in positions:
        e = int(table[b, j // page]) if 0 <= j // page < table.size(1) else -1
        out.append(e * page + j % page if 0 <= e < pages else -1)
    return torch.tensor(out, dtype=torch.int64)


def _write_reference(a, qn, kn, freqs, kv, scale, pe, table, starts, counts, bad=()):
    def norm(x, w):
        r = (1 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
        return (x.float() * r * w.float()).bfloat16().float()
    qr = 0 if qn is None else qn.numel()
    kv, scale, pe = kv.clone(), scale.clone(), pe.clone()
    pages, page = scale.shape
    codes, s = _quantised(norm(a[..., qr:qr + C], kn))
    key = _rotated(a[..., qr + C:], freqs).bfloat16()
    for b in range(a.size(0)):
        if starts[b] < 0:
            continue
        for i, row in enumerate(_rows(table, page, pages, b, range(int(starts[b]), int(starts[b]) + min(int(counts[b]), a.size(1))))):
            if row >= 0:
                kv.view(torch.uint8).view(-1, C)[row] = codes[b, i].view(torch.uint8)
                scale.view(-1)[row], pe.view(-1, ROPE)[row] = s[b, i], key[b, i]
    if qr:
        n = norm(a[..., :qr], qn).unflatten(-1, (-1, 128))
        ys = n.abs().amax(-1).clamp_min(1e-4) / torch.tensor(448.0)
        return kv, scale, pe, (n / ys[..., None]).to(FP8).flatten(-2), ys
    return kv, scale, pe, a.new_empty(*a.shape[:2], 0, dtype=FP8), a.new_empty(*a.shape[:2], 0, dtype=torch.float32)


# one row and many; pages of one group of eight, of no power of two, larger than the sequence; ragged batches, sequences without rows
WRITE = [(1, 1, 1536, 64), (1, 1, 0, 8), (3, 5, 128, 24), (2, 33, 512, 8), (1, 200, 2048, 4096), (65, 3, 0, 16), (4, 7, 0, 40), (1, 1000, 0, 64)]


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
    a[0, 0, qr:qr + C] *= 1e-5                                        # amax below the smallest scale's
    if s > 2:
        a[0, 1, qr + 3], a[0, 2, qr + 77] = float("nan"), float("inf")
    qn = (1 + 0.1 * torch.randn(qr, generator=g)).bfloat16() if qr else None
    kn = (1 + 0.1 * torch.randn(C, generator=g)).bfloat16()
    pool = _pool(g, pages, page)
    freqs = _phases(g, b, s)
    want = _write_reference(a, qn, kn, freqs, *pool, table, starts, counts)
    dev = [t.cuda() for t in pool]
    y, ys = torch.ops.dsv3fp8.mla_latent_paged(a.cuda(), None if qn is None else qn.cuda(), kn.cuda(), freqs.cuda(), *dev, table.cuda(), starts.cuda(), counts.cuda(), EPS, EPS)
    # the same roundings in the same places, the root's sum in binary64: bit for bit
    for got, ref in zip((*dev[:2], dev[2], y, ys), want):
        same = _bits(got) == _bits(ref)
        if got.dtype.is_floating_point and got.element_size() > 1:
            same |= torch.isnan(got.float().cpu()) & torch.isnan(ref.float())
        assert same.all()
    if s > 2:
        bad = _rows(table, page, pages, 0, [38, 39])
        assert torch.isnan(dev[1].view(-1).cpu()[bad]).all() and (_bits(dev[0]).view(-1, C)[bad] == 0).all()


# lengths of nothing, one, a page's end and its neighbours; more positions than the table has pages for
READ = [([0], 1, 8), ([1], 1, 8), ([700], 700, 64), ([7, 8, 9, 0, 64, 63, 65], 70, 24), ([100, 1], 37, 8), ([5, 300], 400, 16), ([-3, 12], 16, 8)]


@pytest.mark.parametrize("lengths,positions,page", READ)
def test_rows_are_read_back(lengths, positions, page):
    g = torch.Generator().manual_seed(positions)
    b, n = len(lengths), [max(0, x) for x in lengths]
    pages = sum(-(-x // page) for x in n) + 1
    table, pool = _tables(g, n, page, pages), _pool(g, pages, page)
    if n[-1] > page:
        table[-1, 1] = -1                                            # a page that the sequence does not have
    pool[1][0, 0] = float("nan")                                     # a row that was not finite
    kv, pe = torch.ops.dsv3fp8.mla_cache_read(*[t.cuda() for t in pool], table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), positions)
    assert kv.shape == (b, positions, C) and pe.shape == (b, positions, ROPE)
    want_kv, want_pe = torch.zeros(b, positions, C), torch.zeros(b, positions, ROPE).bfloat16()
    for i in range(b):
        row = _rows(table, page, pages, i, range(min(n[i], positions)))
        live = (row >= 0).nonzero().flatten()
        want_kv[i, live] = pool[0].view(-1, C)[row[live]].float() * pool[1].view(-1)[row[live], None]
        want_pe[i, live] = pool[2].view(-1, ROPE)[row[live]]
    want = want_kv.bfloat16()
    assert torch.equal(want.nan_to_num(7.0), kv.cpu().nan_to_num(7.0)) and torch.equal(_bits(pe), _bits(want_pe))


@pytest.mark.parametrize("page", [8, 24, 64])
@pytest.mark.parametrize("b,most", [(1, 1), (1, 4), (3, 9), (70, 3), (2, 64)])
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


def test_empty_calls():
    g = torch.Generator().manual_seed(0)
    pool = [t.cuda() for t in _pool(g, 2, 8)]
    none, table = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    kv, pe = torch.ops.dsv3fp8.mla_cache_read(*pool, table, none, 5)
    assert kv.shape == (0, 5, C) and pe.shape == (0, 5, ROPE)
    torch.ops.dsv3fp8.mla_cache_keep(*pool, table, none, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), none)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv, _ = torch.ops.dsv3fp8.mla_cache_read(*pool, one[None], one, 0)
    assert kv.shape == (1, 0, C)
    a = torch.zeros(1, 0, C + ROPE, device="cuda").bfloat16()
    y, ys = torch.ops.dsv3fp8.mla_latent_paged(a, None, torch.ones(C, device="cuda").bfloat16(), torch.zeros(1, 0, 32, dtype=torch.complex64, device="cuda"), *pool,
                                               one[None], one, one, EPS, EPS)
    assert y.shape == (1, 0, 0) and ys.shape == (1, 0, 0)


def test_rows_past_32_bits_of_bytes():
    """A pool of more than 2^32 bytes of codes, pages from its end."""
    page, pages = 4096, 2200
    kv = torch.zeros(pages, page, C, dtype=torch.uint8, device="cuda").view(FP8)
    scale, pe = torch.ones(pages, page, device="cuda"), torch.zeros(pages, page, ROPE, device="cuda").bfloat16()
    assert kv.numel() > 2 ** 32
    g = torch.Generator().manual_seed(3)
    table = torch.tensor([[pages - 1, 7, pages - 2]], dtype=torch.int32)
    a, freqs = torch.randn(1, 9000, C + ROPE, generator=g).bfloat16(), _phases(g, 1, 9000)
    kn = torch.ones(C).bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    torch.ops.dsv3fp8.mla_latent_paged(a.cuda(), None, kn.cuda(), freqs.cuda(), kv, scale, pe, table.cuda(), i32(0), i32(9000), EPS, EPS)
    small = [torch.zeros(3, page, C, dtype=torch.uint8).view(FP8), torch.ones(3, page), torch.zeros(3, page, ROPE).bfloat16()]
    want = _write_reference(a, None, kn, freqs, *small, torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.zeros(1).int(), torch.full((1,), 9000).int())
    for big, ref in zip((kv, scale, pe), want):
        assert torch.equal(_bits(big[[7, pages - 2, pages - 1]]) if big.element_size() > 1 else _bits(big.view(torch.uint8)[[7, pages - 2, pages - 1]]), _bits(ref))
    got_kv, got_pe = torch.ops.dsv3fp8.mla_cache_read(kv, scale, pe, table.cuda(), i32(9000), 9000)
    rows = _rows(torch.tensor([[2, 0, 1]]), page, 3, 0, range(9000))
    assert torch.equal(got_kv[0].cpu(), (want[0].view(-1, C)[rows].float() * want[1].view(-1)[rows, None]).bfloat16())
    assert torch.equal(_bits(got_pe[0]), _bits(want[2].view(-1, ROPE)[rows]))
