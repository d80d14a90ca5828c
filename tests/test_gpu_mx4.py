"""Microscaled 4-bit numbers on the GPU: into the format, back, and products with weights in it, against plain evaluations in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FP8, FP4, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
VALUES = torch.tensor(MAGNITUDES + [-v for v in MAGNITUDES], dtype=torch.float64)


@pytest.fixture(scope="module")
def K():
    import dsv3fp8
    return dsv3fp8


@pytest.fixture(autouse=True)
def _default_dtype():
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(old)


def quantised(x):
    """Codes 0 .. 15 and scale bytes of x [.., k] by search: the exponent upwards until nothing is above 6, the code among all eight."""
    x = x.double().cpu().unflatten(-1, (-1, 32))
    top, fine = x.abs().amax(-1), x.isfinite().all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    e = torch.full(top.shape, -127, dtype=torch.int32)
    for _ in range(254):
        e += (torch.where(fine, top, 0.0) > 6 * torch.exp2(e.double())).int()
    v = (x * torch.exp2(-e.double())[..., None])
    gap = (v.abs()[..., None] - VALUES[:8]).abs()
    # ties to the even code: odd ones count as a trifle further away
    code = (gap + torch.tensor([0.0, 1e-12] * 4, dtype=torch.float64)).argmin(-1)
    code = code | torch.where(torch.signbit(v), 8, 0)
    code = torch.where(fine[..., None], code, 0).flatten(-2)
    return code, torch.where(fine, e + 127, 255).to(torch.uint8)


def packed(code):
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)


def held(y, s):
    """The values of packed codes and scales, in 64 bits."""
    b = y.cpu().view(torch.uint8).long()
    v = VALUES[torch.stack((b & 15, b >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32))
    e = s.cpu().view(torch.uint8).double()
    p = torch.where(e == 255, float("nan"), torch.exp2(e - 127))
    return (v * p[..., None]).flatten(-2)


def numbers(codes, scales, device="cuda"):
    """Tensors of the format from codes 0 .. 15 and bytes."""
    return packed(codes).view(FP4).to(device), scales.to(torch.uint8).view(E8M0).to(device)


# one block, ragged ends of a workgroup's share (1024 eights), three dimensions, long rows
SHAPES = [(32,), (1, 64), (3, 5, 96), (257, 32), (33, 992), (1, 7168), (70, 7168)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantised(K, shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g, dtype=torch.float32) * torch.exp2(torch.randint(-12, 12, shape[:-1] + (shape[-1] // 32,), generator=g).float()).repeat_interleave(32, -1)
    x = x.to(dtype)
    y, s = K.mx4_quant(x.cuda())
    assert y.dtype == FP4 and s.dtype == E8M0 and y.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], shape[-1] // 32)
    code, byte = quantised(x)
    assert torch.equal(s.cpu().view(torch.uint8), byte) and torch.equal(y.cpu().view(torch.uint8), packed(code))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_borders(K, dtype):
    """Largest elements around the steps of the scale, every tie of the codes, the type's smallest and largest numbers, zeros."""
    top = torch.tensor([6.0, 6.03125, 5.96875, 4.0, 3.0, 3.015625, 12.0, 11.9375, 12.0625, 1.5, 1.5078125, 0.75, 0.0, 7.0, 1e-4, 448.0])
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2, 0.3, 0.7, 0.8, 1.3, 1.7, 2.4, 2.6, 3.4, 3.6, 4.9, 5.1, 0.0, -0.0, 0.125, 5.5, 6.0, 4.0])
    rows = [torch.cat([t[None], torch.zeros(31)]) for t in top] + [torch.cat([torch.tensor([6.0]), ties, -ties[:6]])]
    x = torch.stack(rows).float()
    info = torch.finfo(dtype)
    small = info.smallest_normal if dtype != torch.float32 else 2.0 ** -126
    ends = torch.stack([torch.full((32,), v, dtype=torch.float64) for v in (info.max, -info.max, small, small / 2, 4 * small, 6 * small)]
                       + [torch.cat([torch.tensor([info.max], dtype=torch.float64), torch.full((31,), small, dtype=torch.float64)])]).float()
    x = torch.cat([x, -x, x * 2.0 ** 9, x * 2.0 ** -9, ends]).to(dtype)
    y, s = K.mx4_quant(x.cuda())
    code, byte = quantised(x)
    assert torch.equal(s.cpu().view(torch.uint8), byte)
    assert torch.equal(y.cpu().view(torch.uint8), packed(code))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_blocks_that_are_not_finite(K, dtype, bad):
    x = torch.ones(4, 96, dtype=dtype)
    x[1, 40] = bad
    x[3, 95] = bad
    y, s = K.mx4_quant(x.cuda())
    v = K.mx4_dequant(y, s).cpu()
    want = torch.ones(4, 96, dtype=torch.bool)
    want[1, 32:64] = want[3, 64:] = False
    assert torch.equal(v == 1, want) and torch.equal(v.isnan(), ~want)
    assert (y.cpu().view(torch.uint8)[~want[:, ::2]] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_all_numbers(K, dtype):
    """Every code beside every scale."""
    codes = torch.arange(256 * 32).view(256, 32) % 16
    y, s = numbers(codes, torch.arange(256)[:, None])
    torch.set_default_dtype(dtype)
    v = K.mx4_dequant(y, s)
    assert v.dtype == dtype and v.shape == (256, 32)
    want = held(y, s)
    # binary32 and bf16 hold all of them but those of 2^127 times 2 and more, which are infinite there as in a conversion
    assert torch.equal(v.cpu().nan_to_num(7.0), want.to(dtype).nan_to_num(7.0)) and torch.equal(v.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("shape", SHAPES)
def test_back(K, shape):
    g = torch.Generator().manual_seed(len(shape) + shape[-1])
    codes = torch.randint(0, 16, shape, generator=g)
    y, s = numbers(codes, torch.randint(90, 160, (*shape[:-1], shape[-1] // 32), generator=g))
    assert torch.equal(K.mx4_dequant(y, s).cpu(), held(y, s).bfloat16())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_more_than_the_caches_hold(K, dtype):
    """Large tensors go past the caches: what comes out is what their rows give in smaller calls."""
    torch.set_default_dtype(dtype)
    x = (torch.randn(9401, 7200, device="cuda", dtype=torch.float32) * torch.rand(9401, 1, device="cuda", dtype=torch.float32)).to(dtype)
    x[77, 5], x[9400, 7199] = float("nan"), float("inf")
    assert x.numel() * x.element_size() > 128 << 20
    y, s = K.mx4_quant(x)
    v = K.mx4_dequant(y, s)
    for i in range(0, 9401, 1000):
        part, scale = K.mx4_quant(x[i:i + 1000])
        assert torch.equal(y.view(torch.uint8)[i:i + 1000], part.view(torch.uint8)) and torch.equal(s.view(torch.uint8)[i:i + 1000], scale.view(torch.uint8))
        back = K.mx4_dequant(part, scale)
        assert torch.equal(v[i:i + 1000].isnan(), back.isnan()) and torch.equal(v[i:i + 1000].nan_to_num(7.0), back.nan_to_num(7.0))


def operands(g, m, n, k, a8, spread=6):
    """Random numbers of all sizes, and their values in 64 bits."""
    b, b_s = numbers(torch.randint(0, 16, (n, k), generator=g), torch.randint(127 - spread, 127 + spread, (n, k // 32), generator=g))
    if a8:
        a = (torch.randn(m, k, generator=g, dtype=torch.float32) * 40).to(FP8)
        a_s = torch.exp2(torch.randint(-spread, spread, (m, k // 128), generator=g).float())
        va = a.double() * a_s.double().repeat_interleave(128, -1)
        return a.cuda(), a_s.cuda(), b, b_s, va, held(b, b_s)
    a, a_s = numbers(torch.randint(0, 16, (m, k), generator=g), torch.randint(127 - spread, 127 + spread, (m, k // 32), generator=g))
    return a, a_s, b, b_s, held(a, a_s), held(b, b_s)


# streamed: every count of rows that is copied, narrow and wide weights, one to many chunks of 512, shorter last ones, wavefronts with none and with several
PRODUCTS = [(1, 1, 128), (1, 576, 7168), (2, 17, 256), (4, 100, 384), (3, 6200, 512), (5, 40, 640), (16, 100, 384), (16, 6145, 1152), (9, 7168, 4096), (17, 48, 2048),
            (32, 6160, 640), (31, 500, 16384), (33, 33, 640), (64, 512, 1152), (65, 130, 128), (65, 64, 1024), (100, 257, 896), (128, 128, 512), (200, 1000, 512)]
# tiles of 64, 128 and 256 rows, with and without slices of k, odd numbers of steps, ragged rows and columns, columns that are no whole eights
PRODUCTS += [(40, 8200, 8192), (64, 8203, 8320), (33, 20000, 1152), (64, 33000, 128), (300, 2304, 7168), (129, 9000, 2176), (257, 3001, 2304), (300, 7300, 384), (520, 6200, 384),
             (1030, 5000, 640), (1500, 8200, 640), (1537, 8193, 1152), (3000, 4352, 512), (1600, 8448, 128), (513, 2050, 1408)]
# scales fetched from where they lie (k a multiple of 512) and laid out
PRODUCTS += [(70, 20000, 2048), (130, 20001, 2176), (60, 33000, 2048), (50, 33001, 2176)]
# a last round of 256 x 256 in halves, the last of which may have no columns: all of them, some; in one and more bands of rows
PRODUCTS += [(1281, 5200, 640), (1200, 5370, 384), (1800, 9300, 640), (1030, 16500, 256), (4500, 8270, 384)]


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(K, m, n, k, a8):
    """Terms are exact.  Of e4m3 activations the matrix core lines eight terms up at the largest one's exponent and cuts what lies more than 13 bits
    below it: at most seven times 2^-13 of the eight's sum of sizes.  Sums of 32 terms of four bits each are exact (multiples of 1/4 up to 1152, times a
    power of two).  Every further addition is off by 2^-23 of the sum so far at most (cut, not rounded): k / 32 in the instructions, 7 of the eight
    wavefronts' or up to eight slices' sums; s slices, k / 256 of them at most, have k / 32 / s in the instructions and s - 1 behind them, which is less."""
    g = torch.Generator().manual_seed(m * 7 + n + k)
    a, a_s, b, b_s, va, vb = operands(g, m, n, k, a8)
    va, vb = va.cuda(), vb.cuda()
    ref, size = va @ vb.t().contiguous(), va.abs() @ vb.abs().t().contiguous()
    bound = size * (k / 32 + 7) * 2.0 ** -23
    if a8:
        bound = bound + size * 7 * 2.0 ** -13
    torch.set_default_dtype(torch.float32)
    c = K.mx4_gemm(a, a_s, b, b_s)
    assert c.shape == (m, n) and ((c.double() - ref).abs() <= bound).all()
    for dtype in (torch.bfloat16, torch.float16):
        torch.set_default_dtype(dtype)
        assert torch.equal(K.mx4_gemm(a, a_s, b, b_s), c.to(dtype))


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 256), (20, 100, 1024), (90, 140, 384), (300, 600, 512), (60, 9000, 7168), (260, 3000, 2560), (1300, 9000, 640), (1900, 8330, 384)])
def test_products_of_whole_numbers(K, m, n, k, a8):
    """Whole numbers whose sums binary32 holds come out exactly, whatever the order: codes of 0, 1, 2, 3, 4 and 6, scales of 1, 2 and 4."""
    g = torch.Generator().manual_seed(m + n)
    pick = torch.tensor([0, 2, 4, 5, 6, 7, 10, 12, 13, 14, 15])
    b, b_s = numbers(pick[torch.randint(0, 11, (n, k), generator=g)], torch.randint(127, 130, (n, k // 32), generator=g))
    if a8:
        a = torch.randint(-8, 9, (m, k), generator=g).float().to(FP8).cuda()
        a_s = torch.exp2(torch.randint(0, 3, (m, k // 128), generator=g).float()).cuda()
        va = a.double().cpu() * a_s.double().cpu().repeat_interleave(128, -1)
    else:
        a, a_s = numbers(pick[torch.randint(0, 11, (m, k), generator=g)], torch.randint(127, 130, (m, k // 32), generator=g))
        va = held(a, a_s)
    torch.set_default_dtype(torch.float32)
    assert torch.equal(K.mx4_gemm(a, a_s, b, b_s).cpu().double(), va @ held(b, b_s).t())


@pytest.mark.parametrize("k", [640, 1024])
@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n", [(3, 50), (80, 300), (300, 7000), (50, 20000), (1500, 9000), (1900, 8330)])
def test_a_scale_of_nan_reaches_its_row(K, m, n, a8, k):
    g = torch.Generator().manual_seed(m)
    a, a_s, b, b_s, _, _ = operands(g, m, n, k, a8)
    plain = K.mx4_gemm(a, a_s, b, b_s)
    b_s.view(torch.uint8)[n - 2, 7] = 255
    if a8:
        a_s[m - 1, 2] = float("nan")
    else:
        a_s.view(torch.uint8)[m - 1, 19] = 255
    c = K.mx4_gemm(a, a_s, b, b_s)
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[:, n - 2] = nan[m - 1] = True
    assert torch.equal(c.isnan(), nan) and torch.equal(c[~nan], plain[~nan])


@pytest.mark.parametrize("m,n,k,lead", [(0, 64, 128, (0,)), (4, 0, 128, (4,)), (6, 40, 128, (2, 3)), (1, 40, 256, ()), (3, 5, 0, (3,))])
def test_shapes(K, m, n, k, lead):
    """Rows of any number of dimensions, no rows, no columns, no terms."""
    codes, scales = numbers(torch.randint(0, 16, (n, k)), torch.full((n, k // 32), 127))
    a, a_s = K.mx4_quant(torch.randn(*lead, k, device="cuda"))
    c = K.mx4_gemm(a, a_s, codes, scales)
    assert c.shape == (*lead, n)
    ref = held(a, a_s).reshape(m, k) @ held(codes, scales).t()
    assert torch.allclose(c.cpu().double().reshape(m, n), ref, rtol=2.0 ** -8, atol=1e-5)
    y, s = K.mx4_quant(torch.randn(*lead, k, device="cuda"))
    assert K.mx4_dequant(y, s).shape == (*lead, k)


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(5, 40, 384), (300, 700, 384), (300, 7000, 384), (300, 2304, 512)])
def test_rows_of_larger_tensors(K, m, n, k, a8):
    """From the second row on, where scales begin at no more than multiples of four bytes, or of 16."""
    g = torch.Generator().manual_seed(m)
    a, a_s, b, b_s, _, _ = operands(g, m + 1, n + 1, k, a8)
    want = K.mx4_gemm(a[1:].clone(), a_s[1:].clone(), b[1:].clone(), b_s[1:].clone())
    assert torch.equal(K.mx4_gemm(a[1:], a_s[1:], b[1:], b_s[1:]), want)


def test_the_same_sums_in_every_call(K):
    for m in (1, 40, 100, 600):
        g = torch.Generator().manual_seed(m)
        a, a_s, b, b_s, _, _ = operands(g, m, 7000, 4096, m % 3 == 0)
        first = K.mx4_gemm(a, a_s, b, b_s)
        for _ in range(3):
            assert torch.equal(K.mx4_gemm(a, a_s, b, b_s), first)


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m", [1, 50, 300])
def test_captured_and_replayed(K, m, a8):
    """Quantise and multiply in a graph, replayed on new contents between eager calls."""
    g = torch.Generator().manual_seed(m)
    n, k = 9000, 4096
    _, _, b, b_s, _, _ = operands(g, m, n, k, a8)
    x = torch.randn(m, k, generator=g, dtype=torch.float32).bfloat16().cuda()

    def step():
        a, a_s = K.act_quant(x, 128, "ue8m0") if a8 else K.mx4_quant(x)
        return K.mx4_gemm(a, a_s, b, b_s), K.mx4_dequant(*K.mx4_quant(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.copy_(torch.randn(m, k, generator=g, dtype=torch.float32).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_streams_at_once(K):
    sets = []
    for seed, m in ((1, 200), (2, 300)):
        g = torch.Generator().manual_seed(seed)
        a, a_s, b, b_s, _, _ = operands(g, m, 3000, 4096, seed == 1)
        sets.append((a, a_s, b, b_s))
    want = [K.mx4_gemm(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(K.mx4_gemm(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(c, want[i]) for i in range(2) for c in got[i])


def test_past_32_bits_of_elements(K):
    """2^31 elements and more: their ends are what the last rows give by themselves."""
    x = torch.randn(300001, 7168, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    y, s = K.mx4_quant(x)
    last, scale = K.mx4_quant(x[-9:].contiguous())
    assert torch.equal(y[-9:].view(torch.uint8), last.view(torch.uint8)) and torch.equal(s[-9:].view(torch.uint8), scale.view(torch.uint8))
    torch.set_default_dtype(torch.bfloat16)
    assert torch.equal(K.mx4_dequant(y, s)[-9:], K.mx4_dequant(last, scale))


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(3, 700001, 16384), (40, 700001, 16384), (4001, 600011, 256), (70001, 40, 128)])
def test_products_past_32_bits_of_bytes(K, m, n, k, a8):
    """Weights of more than 2^32 bytes, results of more than 2^31 elements: exact sums, so that the last rows and columns are those of a product of their own."""
    g = torch.Generator(device="cuda").manual_seed(m)
    b = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8).view(FP4)
    b_s = torch.full((n, k // 32), 127, device="cuda", dtype=torch.uint8).view(E8M0)
    if a8:
        a, a_s = torch.randint(-8, 9, (m, k), generator=g, device="cuda").float().to(FP8), torch.ones(m, k // 128, device="cuda", dtype=torch.float32)
    else:
        a = torch.randint(0, 256, (m, k // 2), generator=g, device="cuda", dtype=torch.uint8).view(FP4)
        a_s = torch.full((m, k // 32), 127, device="cuda", dtype=torch.uint8).view(E8M0)
    c = K.mx4_gemm(a, a_s, b, b_s)
    assert c.shape == (m, n)
    rows, cols = min(m, 3), min(n, 300)
    ends = K.mx4_gemm(a[-rows:].contiguous(), a_s[-rows:].contiguous(), b[-cols:].contiguous(), b_s[-cols:].contiguous())
    first = K.mx4_gemm(a[:rows].contiguous(), a_s[:rows].contiguous(), b[:cols].contiguous(), b_s[:cols].contiguous())
    assert torch.equal(c[-rows:, -cols:], ends) and torch.equal(c[:rows, :cols], first)


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n", [(2097120, 5), (2097121, 9), (4194250, 16)])
def test_no_terms_and_more_rows_than_a_launch_holds(K, m, n, a8):
    """k == 0: zeros, for any number of rows."""
    b, b_s = torch.empty(n, 0, dtype=torch.uint8, device="cuda").view(FP4), torch.empty(n, 0, dtype=torch.uint8, device="cuda").view(E8M0)
    a = torch.empty(m, 0, dtype=torch.uint8, device="cuda").view(FP8 if a8 else FP4)
    a_s = torch.empty(m, 0, dtype=torch.float32, device="cuda") if a8 else torch.empty(m, 0, dtype=torch.uint8, device="cuda").view(E8M0)
    for dtype in (torch.bfloat16, torch.float32):
        torch.set_default_dtype(dtype)
        spoilt = torch.full((m * n,), 7.0, dtype=dtype, device="cuda")
        del spoilt                                                  # (what the result's memory holds beforehand)
        c = K.mx4_gemm(a, a_s, b, b_s)
        assert c.shape == (m, n) and c.dtype == dtype and (c == 0).all()


@pytest.mark.parametrize("a8", [False, True], ids=["mx4", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 640), (20, 70, 512), (40, 300, 1152), (70, 8200, 512), (300, 700, 640), (1030, 5000, 640)])
def test_products_of_scales_at_both_ends(K, m, n, k, a8):
    """Scales of 2^-127 beside scales of 2^127, block by block, so that every product is an ordinary number; the bound is `test_product`'s.  (Activations' e4m3 scales
    are powers of two that binary32 has as normal numbers.)"""
    g = torch.Generator().manual_seed(m + k)
    ends = torch.tensor([0, 1, 2, 3, 60, 127, 190, 251, 252, 253, 254])
    pick = ends[torch.randint(0, 11, (k // 128,), generator=g)] if a8 else ends[torch.randint(0, 11, (k // 32,), generator=g)]
    if a8:
        pick = pick.clamp(1, 253)
        a = (torch.randn(m, k, generator=g, dtype=torch.float32) * 40).to(FP8)
        a_s = torch.exp2(pick.double() - 127).float().expand(m, -1).contiguous()
        va = a.double() * a_s.double().repeat_interleave(128, -1)
        a, a_s, other = a.cuda(), a_s.cuda(), (254 - pick).repeat_interleave(4)
    else:
        a, a_s = numbers(torch.randint(0, 16, (m, k), generator=g), pick.expand(m, -1))
        va, other = held(a, a_s), 254 - pick
    b, b_s = numbers(torch.randint(0, 16, (n, k), generator=g), other.expand(n, -1))
    vb = held(b, b_s)
    ref, size = va @ vb.t(), va.abs() @ vb.abs().t()
    bound = size * (k / 32 + 7) * 2.0 ** -23 + (size * 7 * 2.0 ** -13 if a8 else 0)
    torch.set_default_dtype(torch.float32)
    c = K.mx4_gemm(a, a_s, b, b_s).cpu().double()
    assert ref.abs().max() > 1 and ((c - ref).abs() <= bound).all()


@pytest.mark.parametrize("m,n,k", [(1, 40, 640), (40, 300, 1152), (300, 700, 640), (1030, 5000, 640)])
def test_products_smaller_and_larger_than_binary32(K, m, n, k):
    """Scales of 2^-127 on both sides: zeros.  Of 2^127 on both: infinities of the sums' sign where all terms have one sign."""
    torch.set_default_dtype(torch.float32)
    a, _ = numbers(torch.full((m, k), 7), torch.zeros(m, k // 32))
    codes = torch.full((n, k), 7)
    codes[1::2] = 15
    b, _ = numbers(codes, torch.zeros(n, k // 32))
    scales = lambda rows, byte: torch.full((rows, k // 32), byte, dtype=torch.uint8).cuda().view(E8M0)  # noqa: E731
    assert (K.mx4_gemm(a, scales(m, 0), b, scales(n, 0)) == 0).all()
    c = K.mx4_gemm(a, scales(m, 254), b, scales(n, 254))
    assert (c[:, 0::2] == float("inf")).all() and (c[:, 1::2] == float("-inf")).all()
