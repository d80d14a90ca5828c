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


# ------------------------------------------------------------------------------------------------------------ attention

def _bits_of(rows):
    """[batch][nodes] sets of nodes -> int64 [batch, nodes]."""
    out = [[sum(1 << j for j in seen) for seen in seq] for seq in rows]
    return torch.tensor([[v - (1 << 64) if v >> 63 else v for v in seq] for seq in out], dtype=torch.int64)


def _trees(kind, g, b, s):
    """What each new token sees of the new ones: None (those in front of it and itself), ancestors of a random tree, any bits (the
    second token none)."""
    if kind is None:
        return None, [[set(range(i + 1)) for i in range(s)] for _ in range(b)]
    rows = []
    for _ in range(b):
        seq = []
        for i in range(s):
            if kind == "any":
                seq.append(set((torch.rand(s, generator=g) < 0.4).nonzero().flatten().tolist()) if i != 1 else set())
            else:
                parent = int(torch.randint(max(0, i - 5), i, (1,), generator=g)) if i else None
                seq.append(({i} | seq[parent]) if i else {0})
        rows.append(seq)
    return _bits_of(rows), rows


def _attention_case(b, s, h, context, page, kind, seed):
    """Sequences of uneven lengths (the first the longest, the second with no more than the new tokens), fewer tokens in some, NaN in the
    queries of tokens that a sequence does not have and in the cache rows behind every sequence."""
    g = torch.Generator().manual_seed(seed)
    lengths = [context] + [s + int(torch.randint(0, max(1, context - s + 1), (1,), generator=g)) for _ in range(b - 1)]
    counts = [s] + [int(torch.randint(0, s + 1, (1,), generator=g)) for _ in range(b - 1)]
    if b > 1:
        lengths[1], counts[1] = s, s
    if b > 3:
        counts[3] = 0
    starts = [n - s for n in lengths]
    pages = sum(-(-n // page) for n in lengths) + 1
    table, pool = _tables(g, lengths, page, pages), _pool(g, pages, page)
    nan = torch.full((pages * page,), True)
    for i in range(b):
        nan[_rows(table, page, pages, i, range(starts[i] + counts[i]))] = False
    pool[0].view(torch.uint8).view(-1, C)[nan] = 0x7f
    pool[2].view(-1, ROPE)[nan] = float("nan")
    q = (torch.randn(b, s, h, NOPE + ROPE, generator=g) * 2).bfloat16()
    for i in range(b):
        q[i, counts[i]:] = float("nan")
    bits, seen = _trees(kind, g, b, s)
    w8 = torch.randn(h * (NOPE + V), C, generator=g).to(FP8)
    ws = torch.rand(h * 2, C // 128, generator=g) * 0.03 + 0.01
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    args = [q, _phases(g, b, s), *pool, table, i32(starts), i32(counts), bits, w8, ws, context, 0.08]
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in args], seen


def _attention_reference(args, seen):
    """Binary64 with the roundings to bf16 that the weights and the rotated query have."""
    q, freqs, kv, scale, pe, table, starts, counts, _, w8, ws, positions, softmax_scale = args
    b, s, h, _ = q.shape
    pages, page = scale.shape
    w = (w8.float() * ws.repeat_interleave(128, 0).repeat_interleave(128, 1)).bfloat16().double().view(h, NOPE + V, C)
    out = torch.zeros(b, s, h, V, dtype=torch.float64, device=q.device)
    for i in range(b):
        first, n = int(starts[i]), int(counts[i])
        if n <= 0 or first < 0:
            continue
        end = min(first + n, positions)
        rows = _rows(table.cpu(), page, pages, i, range(end))
        visible = torch.zeros(n, end, dtype=torch.bool)
        visible[:, :first] = True
        for t in range(n):
            for j in seen[i][t]:
                if first + j < end:
                    visible[t, first + j] = True
        visible &= (rows >= 0)[None]
        used = rows.clamp_min(0).cuda()
        there = (rows >= 0).cuda()[:, None]
        c = torch.where(there, kv.view(-1, C)[used].double() * scale.view(-1)[used, None].double(), 0.0)
        k = torch.where(there, pe.view(-1, ROPE)[used].double(), 0.0)
        turned = _rotated(q[i, :n, :, NOPE:], freqs[i, :n, None]).bfloat16().double()
        visible = visible.cuda()
        for a in range(h):
            folded = q[i, :n, a, :NOPE].double() @ w[a, :NOPE]
            score = (folded @ c.T + turned[:, a] @ k.T) * softmax_scale
            p = score.masked_fill(~visible, float("-inf")).softmax(-1).masked_fill(~visible, 0)
            for t in range(n):              # (a product with a weight of zero would bring in what the token does not see)
                if bool(visible[t].any()):
                    out[i, t, a] = (p[t, visible[t]] @ c[visible[t]]) @ w[a, NOPE:].T
    return out


def _close(got, ref):
    # The latent sum and the result round to bf16 (2^-8 of the value at most each: 2^-8 of the norm for the result, as much for the sum, whose errors
    # a random product of 512 terms carries over in proportion); folded queries and exponentials are pairs of codes, 2^-9 at most, which
    # average out over 512 features and the positions: 2^-7 of the row's norm
    return ((got - ref).norm(dim=-1) <= 2.0 ** -7 * ref.norm(dim=-1)).all()


# one token and 64; heads that fill no block of rows; contexts of one tile and many, of nothing but the new tokens; pages that end inside a
# tile, hold a tile, hold everything; more sequences than compute units, more row blocks than compute units
ATTEND = [(1, 1, 1, 1, 8, None), (1, 1, 128, 31, 64, None), (2, 1, 128, 33, 8, None), (1, 1, 128, 700, 64, None), (5, 1, 16, 1000, 24, None),
          (70, 1, 128, 97, 16, None), (6, 5, 40, 257, 40, None), (3, 64, 3, 64, 8, "tree"), (2, 25, 128, 300, 24, "tree"), (4, 13, 20, 500, 64, "any"),
          (1, 61, 128, 1500, 128, "tree"), (1, 1, 3, 9000, 4096, None), (300, 1, 4, 60, 8, None), (5, 64, 70, 90, 8, "any"), (1, 40, 100, 40, 48, "any"),
          (9, 2, 64, 333, 16, "tree"), (20, 1, 16, 3000, 32, None), (130, 3, 64, 200, 64, "tree"), (1, 2, 32, 64, 64, None)]


# up to 32 (token, head) rows a sequence, whose positions the wavefronts share: none for some of them, many, several tokens, heads that do not divide 32
ATTEND += [(2, 8, 4, 300, 24, "tree"), (3, 16, 2, 700, 64, "any"), (2, 32, 1, 130, 8, "tree"), (1, 1, 32, 128, 16, None), (1, 1, 32, 129, 16, None),
           (4, 2, 16, 5000, 40, None), (7, 3, 10, 260, 64, "any"), (1, 1, 33, 500, 64, None), (600, 1, 16, 40, 8, None), (2, 1, 16, 20000, 64, None)]


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("b,s,h,context,page,kind", ATTEND)
def test_attention(b, s, h, context, page, kind, grow):
    args, seen = _attention_case(b, s, h, context, page, kind, b + s + context)
    if grow:                    # scores that grow along the positions by far more than 2^64: the running maximum is raised
        if kind is not None or context < 8:
            pytest.skip("one run per shape without a tree")
        for i in range(b):
            n = int(args[6][i] + args[7][i])
            rows = _rows(args[5].cpu(), page, args[3].size(0), i, range(n)).cuda()
            args[4].view(-1, ROPE)[rows] *= torch.linspace(0.01, 400, n, device="cuda").bfloat16()[:, None]
    got = torch.ops.dsv3fp8.mla_decode_paged(*args).view(b, s, h, V).double()
    ref = _attention_reference(args, seen)
    assert torch.isfinite(got).all()
    for i in range(b):
        assert (got[i, max(0, int(args[7][i])):] == 0).all()
    if kind == "any" and args[6].min() == 0:
        i = int((args[6] == 0).nonzero()[0])
        assert (got[i, 1] == 0).all()                               # a token that sees nothing
    assert _close(got, ref)


@pytest.mark.parametrize("b,s,h,context,page,kind", [(1, 1, 128, 33, 64, None), (1, 1, 8, 8192, 64, None), (3, 13, 24, 200, 24, "any"), (37, 1, 128, 70, 8, None), (2, 9, 128, 200, 40, "tree")])
def test_attention_quantised_is_the_rounded_result_quantised(b, s, h, context, page, kind):
    from dsv3fp8 import kernel
    args, _ = _attention_case(b, s, h, context, page, kind, 5)
    y = torch.ops.dsv3fp8.mla_decode_paged(*args)
    yq, ys = torch.ops.dsv3fp8.mla_decode_paged_quant(*args)
    rq, rs = kernel.act_quant(y)
    assert torch.equal(yq.view(torch.uint8), rq.view(torch.uint8)) and torch.equal(ys.view(torch.int32), rs.view(torch.int32))
    assert torch.equal(_bits(y), _bits(torch.ops.dsv3fp8.mla_decode_paged(*args)))          # and the same again


@pytest.mark.parametrize("h,page", [(128, 64), (6, 24), (2, 40)])
def test_rows_that_are_not_finite_reach_those_who_see_them(h, page):
    """A latent of NaN (stored as zeros and a scale of NaN) and a key of NaN or infinity, in a drafted branch: the tokens of other branches do
    not notice; then one in the context, which everybody sees."""
    args, seen = _attention_case(2, 12, h, 150, page, "tree", 11)
    clean = torch.ops.dsv3fp8.mla_decode_paged(*args)
    first, pages = int(args[6][0]), args[3].size(0)
    row = lambda j: int(_rows(args[5].cpu(), page, pages, 0, [j])[0])  # noqa: E731
    for what in ("latent", "nan key", "inf key"):
        node = 7
        kv, scale, pe = args[2].clone(), args[3].clone(), args[4].clone()
        if what == "latent":
            kv.view(torch.uint8).view(-1, C)[row(first + node)] = 0
            scale.view(-1)[row(first + node)] = float("nan")
        else:
            pe.view(-1, ROPE)[row(first + node), 3] = float("nan" if what == "nan key" else "inf")
        got = torch.ops.dsv3fp8.mla_decode_paged(args[0], args[1], kv, scale, pe, *args[5:])
        for t in range(12):
            if node in seen[0][t]:
                if what != "inf key":           # (an infinite score of the wrong sign only leaves the others)
                    assert torch.isnan(got[0, t]).all()
            else:
                assert torch.equal(_bits(got[0, t]), _bits(clean[0, t]))
        assert torch.equal(_bits(got[1]), _bits(clean[1]))
    kv, scale = args[2].clone(), args[3].clone()
    kv.view(torch.uint8).view(-1, C)[row(3)] = 0
    scale.view(-1)[row(3)] = float("nan")
    got = torch.ops.dsv3fp8.mla_decode_paged(args[0], args[1], kv, scale, *args[4:])
    assert torch.isnan(got[0]).all() and torch.equal(_bits(got[1]), _bits(clean[1]))


@pytest.mark.parametrize("h", [20, 8])
@pytest.mark.parametrize("page", [8, 40, 64])
def test_attention_skips_what_is_no_page(page, h):
    args, seen = _attention_case(3, 4, h, 230, page, "tree", 2)
    pages = args[3].size(0)
    for i, k, entry in ((0, 1, -1), (0, 2, pages), (2, 0, 2 ** 31 - 1), (1, 0, -7)):
        if k < args[5].size(1):
            args[5][i, k] = entry
    got = torch.ops.dsv3fp8.mla_decode_paged(*args).view(3, 4, h, V).double()
    assert torch.isfinite(got).all() and _close(got, _attention_reference(args, seen))


def test_attention_past_the_stated_positions_and_negative_starts():
    args, seen = _attention_case(4, 3, 16, 200, 16, None, 4)
    args[11] = 150                                                  # the longest sequence is cut there
    args[6][2] = -5                                                 # nothing
    got = torch.ops.dsv3fp8.mla_decode_paged(*args).view(4, 3, 16, V).double()
    assert (got[2] == 0).all() and torch.isfinite(got).all()
    assert _close(got, _attention_reference(args, seen))


def test_attention_of_nobody():
    args, _ = _attention_case(3, 4, 16, 50, 16, "tree", 4)
    args[7].zero_()
    assert (torch.ops.dsv3fp8.mla_decode_paged(*args) == 0).all()
    args, _ = _attention_case(1, 1, 16, 50, 16, None, 4)
    args[0], args[1], args[5], args[6], args[7] = (args[k][:0] for k in (0, 1, 5, 6, 7))
    assert torch.ops.dsv3fp8.mla_decode_paged(*args).shape == (0, 1, 16 * V)


@pytest.mark.parametrize("b,s,h,context", [(3, 1, 128, 500), (2, 20, 16, 300), (3, 2, 16, 700)])
def test_a_step_captured_and_replayed(b, s, h, context):
    """Rows written, attended to and kept in one graph, on a stream of its own; two graphs; lengths, pages and queries change between replays."""
    cases = [_attention_case(b, s, h, context, 24, "tree" if s > 1 else None, seed)[0] for seed in (1, 2, 3)]
    pages = max(c[3].size(0) for c in cases)
    def padded(c):
        c = list(c)
        for k in (2, 3, 4):
            t = c[k]
            big = torch.zeros(pages, *t.shape[1:], dtype=torch.uint8 if k == 2 else t.dtype, device="cuda")
            big[:t.size(0)] = t.view(torch.uint8) if k == 2 else t
            c[k] = big.view(FP8) if k == 2 else big
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

    def fresh(c):
        return [t.clone() if isinstance(t, torch.Tensor) else t for t in c]
    want = []
    for c, rows in zip(cases, a):
        c = fresh(c)
        want.append([t.clone() for t in (*step(c, rows), c[2].view(torch.uint8), c[3], c[4])])
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
                    t.copy_(new) if t.dtype != FP8 else t.view(torch.uint8).copy_(new.view(torch.uint8))
            live_a.copy_(a[k])
            graph.replay()
            torch.ops.dsv3fp8.mla_decode_paged(*cases[k])           # eager work between the replays
        for _, live, _, out in graphs:
            for got, ref in zip((*out, live[2].view(torch.uint8), live[3], live[4]), want[k]):
                assert torch.equal(_bits(got), _bits(ref))


def test_two_streams_at_once():
    one, seen1 = _attention_case(8, 1, 128, 900, 64, None, 21)
    two, seen2 = _attention_case(3, 20, 16, 400, 24, "tree", 22)
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


@pytest.mark.parametrize("h", [16, 8])
def test_attention_past_32_bits_of_bytes(h):
    page, pages = 4096, 2200
    args, seen = _attention_case(2, 3, h, 9000, page, "tree", 6)
    small = args[3].size(0)
    kv = torch.zeros(pages, page, C, dtype=torch.uint8, device="cuda")
    scale, pe = torch.ones(pages, page, device="cuda"), torch.zeros(pages, page, ROPE, device="cuda").bfloat16()
    want = torch.ops.dsv3fp8.mla_decode_paged(*args)
    kv[pages - small:], scale[pages - small:], pe[pages - small:] = args[2].view(torch.uint8), args[3], args[4]
    table = torch.where((args[5] >= 0) & (args[5] < small), args[5] + (pages - small), -1).int()
    got = torch.ops.dsv3fp8.mla_decode_paged(*args[:2], kv.view(FP8), scale, pe, table, *args[6:])
    assert torch.equal(_bits(got), _bits(want)) and _close(got.view(2, 3, h, V).double(), _attention_reference(args, seen))


@pytest.mark.parametrize("order", ["any", "rising", "late"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [17, 25, 60, 118])
@pytest.mark.parametrize("b,s,h,context", [(2, 1, 128, 700), (2, 1, 16, 1500), (1, 9, 40, 300)])
def test_attention_of_scores_of_any_size(b, s, h, context, power, sign, order):
    """Scores of whole numbers times 2^power, formed exactly, up to 2^125: the largest one's positions have all the weight, those of equal ones in equal parts."""
    args, seen = _attention_case(b, s, h, context, 64, "tree" if s > 1 else None, 31)
    args[0].zero_()
    args[0][..., NOPE] = 2.0 ** min(power, 60)
    args[1].fill_(1)
    g = torch.Generator().manual_seed(power)
    for i in range(b):
        n = int(args[6][i] + args[7][i])
        rows = _rows(args[5].cpu(), 64, args[3].size(0), i, range(n)).cuda()
        v = torch.randint(1, 200, (n,), generator=g).float() * sign
        if order == "rising":
            v = v.sort().values
        v *= 2.0 ** max(0, power - 60)
        if order == "late":
            v[:n // 2] *= 2.0 ** -40                             # ordinary scores, then large ones
        args[4].view(-1, ROPE)[rows] = 0
        args[4].view(-1, ROPE)[rows, 0] = v.bfloat16().cuda()
    args[12] = 0.5
    got = torch.ops.dsv3fp8.mla_decode_paged(*args).view(b, s, h, V).double()
    assert torch.isfinite(got).all() and _close(got, _attention_reference(args, seen))


@pytest.mark.parametrize("s,h", [(3, 40), (4, 8)])
def test_counts_out_of_range(s, h):
    """A count above the rows is all rows, a negative one none."""
    args, seen = _attention_case(4, s, h, 200, 24, None, 17)
    args[0] = args[0].nan_to_num(1.0)
    most = 2 ** 31 - 1
    first = args[6].tolist()
    args[6] = torch.tensor([first[0], 0, first[2], most], dtype=torch.int32, device="cuda")
    args[7] = torch.tensor([s, s, 0, s], dtype=torch.int32, device="cuda")
    want = torch.ops.dsv3fp8.mla_decode_paged(*args)
    args[7] = torch.tensor([most, s + 1, -most - 1, most], dtype=torch.int32, device="cuda")
    got = torch.ops.dsv3fp8.mla_decode_paged(*args)
    assert torch.equal(_bits(got), _bits(want)) and (got[2] == 0).all()
