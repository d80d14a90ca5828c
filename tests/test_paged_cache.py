"""The latent cache in pages, on the host: where a position lies, and what its functions refuse (no kernel runs)."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from test_abi import A16, _gpu_body

CSRC = Path(__file__).resolve().parent.parent / "deepseek-v3_amd" / "csrc"
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    from dsv3fp8 import _lib
    return _lib


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    """csrc/paged.hpp, which the kernels use, compiled for the host."""
    at = tmp_path_factory.mktemp("paged")
    (at / "walk.cpp").write_text('#include "paged.hpp"\n'
                                 'extern "C" int64_t row(const int32_t* e, int64_t w, int64_t n, int p, int64_t at) { return dsv3::page_row(e, w, n, p, at); }\n'
                                 'extern "C" void span(int s, int c, int r, int m, int* o) { auto x = dsv3::seq_span(s, c, r, m); o[0] = x.start; o[1] = x.end; o[2] = x.count; }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(at / "walk.cpp"), "-o", str(at / "walk.so")], check=True)
    lib = ctypes.CDLL(str(at / "walk.so"))
    lib.row.restype = ctypes.c_int64
    lib.row.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int64]
    lib.span.argtypes = [ctypes.c_int] * 4 + [ctypes.c_void_p]
    return lib


@pytest.mark.parametrize("page", [8, 24, 64, 16384])
def test_row_of_a_position(walk, page):
    pages = 2 ** 31 // page                                  # rows past 2^31, bytes past 2^40
    table = torch.tensor([3, pages - 1, -1, pages, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32)
    for pos in [0, 1, page - 1, page, page + 7, 2 * page - 1, 2 * page, 3 * page + 5, 4 * page, 5 * page + 1, 6 * page, 7 * page - 1]:
        e = int(table[pos // page])
        want = e * page + pos % page if 0 <= e < pages else -1
        assert walk.row(table.data_ptr(), 7, pages, page, pos) == want
    for pos in [-1, -2 ** 31, 7 * page, 2 ** 31 - 1 + 64, 2 ** 40]:         # in front of the sequence, behind its table
        assert walk.row(table.data_ptr(), 7, pages, page, pos) == -1


def test_span_of_a_sequence(walk):
    o = (ctypes.c_int * 3)()
    for (start, count, rows, most), want in {(5, 3, 4, 100): (5, 8, 3), (-4, 3, 4, 100): (0, 0, 0), (5, -1, 4, 100): (0, 0, 0), (5, 9, 4, 100): (5, 9, 4),
                                             (98, 4, 4, 100): (98, 100, 4), (2 ** 31 - 1, 4, 4, 100): (100, 100, 4), (0, 0, 4, 100): (0, 0, 0),
                                             (-2 ** 31, -2 ** 31, 64, 8388607): (0, 0, 0), (0, 2 ** 31 - 1, 64, 8388607): (0, 64, 64)}.items():
        walk.span(start, count, rows, most, o)
        assert tuple(o) == want


def _cache(L, **change):
    c = dict(kv=A16, kv_scale=A16, pe=A16, pages=4, page_size=64, table=A16, table_width=2) | change
    return ctypes.byref(L.MlaPages(*c.values()))


BAD_PAGES = [({"kv": None}, 1), ({"kv_scale": None}, 1), ({"pe": None}, 1), ({"table": None}, 1), ({"pages": 0}, 2), ({"pages": 2 ** 31}, 2),
             ({"page_size": 0}, 2), ({"page_size": 12}, 2), ({"page_size": 4}, 2), ({"page_size": 16392}, 2), ({"table_width": 0}, 2),
             ({"table_width": 2 ** 31}, 2), ({"kv": A16 + 8}, 4), ({"pe": A16 + 8}, 4), ({"kv_scale": A16 + 2}, 4), ({"table": A16 + 2}, 4)]


def test_latent_paged_validation(L):
    def call(a=A16, stride=2112, qw=A16, kw=A16, f=A16, cache=_cache(L), st=A16, n=A16, y=A16, s=A16, b=2, rows=3, qr=1536, c=512, rope=64):
        return L.lib.dsv3_mla_latent_paged(a, stride, qw, kw, f, cache, st, n, y, s, b, rows, qr, c, rope, 1e-6, 1e-6, None)
    for change, code in BAD_PAGES:
        assert call(cache=_cache(L, **change)) == code
    assert call(cache=None) == 1
    for name in ("a", "qw", "kw", "f", "st", "n", "y", "s"):
        assert call(**{name: None}) == 1 and call(**{name: A16 + 2}) == 4
    for bad in (dict(stride=2104), dict(stride=2113), dict(b=-1), dict(b=65536), dict(rows=-1), dict(rows=1 << 23), dict(b=65535, rows=1 << 16), dict(qr=-128),
                dict(qr=64), dict(qr=2176), dict(c=256), dict(rope=32)):
        assert call(**bad) == 2
    assert call(b=0, a=None) == 0 and call(rows=0, a=None) == 0
    assert call(qr=0, qw=None, y=None, s=None, a=None) == 1          # no query latent: its pointers are not looked at


def test_cache_read_validation(L):
    def call(cache=_cache(L), n=A16, kv=A16, pe=A16, b=2, t=100):
        return L.lib.dsv3_mla_cache_read(cache, n, kv, pe, b, t, None)
    for change, code in BAD_PAGES:
        assert call(cache=_cache(L, **change)) == code
    for name in ("n", "kv", "pe"):
        assert call(**{name: None}) == 1 and call(**{name: A16 + 2}) == 4
    for bad in (dict(b=-1), dict(b=65536), dict(t=-1), dict(t=1 << 23)):
        assert call(**bad) == 2
    assert call(b=0, n=None) == 0 and call(t=0, n=None) == 0


def test_cache_keep_validation(L):
    def call(cache=_cache(L), st=A16, path=A16, kept=A16, b=2, most=5):
        return L.lib.dsv3_mla_cache_keep(cache, st, path, kept, b, most, None)
    for change, code in BAD_PAGES:
        assert call(cache=_cache(L, **change)) == code
    for name in ("st", "path", "kept"):
        assert call(**{name: None}) == 1 and call(**{name: A16 + 2}) == 4
    for bad in (dict(b=-1), dict(b=65536), dict(most=-1), dict(most=65)):
        assert call(**bad) == 2
    assert call(b=0, st=None) == 0 and call(most=0, st=None) == 0


def test_decode_paged_validation(L):
    base = dict(q=A16, f=A16, cache=_cache(L), st=A16, n=A16, tree=A16, w=A16, w_s=A16, y=A16, b=2, rows=3, pos=100, heads=4, nope=128, rope=64, v=128, c=512,
                scale=0.1, ws=0x1000, wsb=1 << 30)
    need = L.lib.dsv3_mla_decode_paged_workspace_bytes(2, 3, 4)
    assert need > 0 and L.lib.dsv3_mla_decode_paged_workspace_bytes(0, 3, 4) == 0

    def plain(**change):
        a = base | change
        return L.lib.dsv3_mla_decode_paged(*[a[k] for k in list(base)[:9]], *[a[k] for k in list(base)[9:]], None)

    def quant(s=A16, **change):
        a = base | change
        return L.lib.dsv3_mla_decode_paged_quant(*[a[k] for k in list(base)[:9]], s, *[a[k] for k in list(base)[9:]], None)
    for call in (plain, quant):
        for change, code in BAD_PAGES:
            assert call(cache=_cache(L, **change)) == code
        for name in ("q", "f", "st", "n", "w", "w_s", "y"):
            assert call(**{name: None}) == 1 and call(**{name: A16 + 2}) == 4
        assert call(tree=A16 + 4) == 4 and call(cache=None) == 1
        for bad in (dict(b=-1), dict(b=65536), dict(rows=-1), dict(rows=65), dict(heads=-1), dict(heads=65536), dict(pos=0), dict(pos=129), dict(nope=64), dict(rope=32),
                    dict(v=64), dict(c=256), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-40)):
            assert call(**bad) == 2, bad
        assert call(cache=_cache(L, table_width=1 << 20), pos=1 << 23) == 2
        assert call(b=65535, cache=_cache(L, table_width=1 << 20), pos=(1 << 23) - 1) == 2        # tiles of all sequences past 31 bits
        assert call(ws=None) == 6 and call(ws=0x1010) == 6 and call(wsb=need - 1) == 6
        assert call(b=0, q=None) == 0 and call(rows=0, q=None) == 0 and call(heads=0, q=None) == 0
    assert quant(s=None) == 1 and quant(s=A16 + 2) == 4


def _args(name):
    z = torch.zeros
    i32 = dict(dtype=torch.int32)
    cache = [z(4, 16, 512, dtype=FP8), z(4, 16), z(4, 16, 64, dtype=torch.bfloat16), z(2, 3, **i32)]
    if name == "mla_latent_paged":
        return [z(2, 3, 128 + 576, dtype=torch.bfloat16), z(128, dtype=torch.bfloat16), z(512, dtype=torch.bfloat16), z(2, 3, 32, dtype=torch.complex64), *cache,
                z(2, **i32), z(2, **i32), 1e-6, 1e-6]
    if name == "mla_cache_read":
        return [*cache, z(2, **i32), 20]
    if name == "mla_cache_keep":
        return [*cache, z(2, **i32), z(2, 5, **i32), z(2, **i32)]
    return [z(2, 3, 4, 192, dtype=torch.bfloat16), z(2, 3, 32, dtype=torch.complex64), *cache, z(2, **i32), z(2, **i32), z(2, 3, dtype=torch.int64),
            z(1024, 512, dtype=FP8), z(8, 4), 20, 0.1]


# where the cache stands, and the int32 [batch] behind it
OPERATORS = {"mla_latent_paged": (4, (8, 9)), "mla_cache_read": (0, (4,)), "mla_cache_keep": (0, (4, 6)), "mla_decode_paged": (2, (6, 7)), "mla_decode_paged_quant": (2, (6, 7))}


@pytest.mark.parametrize("name", OPERATORS)
def test_operators_refuse_tensors_of_two_devices(name):
    with pytest.raises(RuntimeError, match="on the GPU"):
        _gpu_body(name, *_args(name))
    for at, t in enumerate(_args(name)):
        if isinstance(t, torch.Tensor):
            args = _args(name)
            args[at] = t.to("meta")
            with pytest.raises(RuntimeError, match="one device"):
                _gpu_body(name, *args)


@pytest.mark.parametrize("name", OPERATORS)
def test_operators_refuse_what_their_kernels_cannot_read(name):
    at, ints = OPERATORS[name]
    z = torch.zeros
    bad = {at: [lambda t: t.bfloat16(), lambda t: t[:0], lambda t: z(4, 12, 512, dtype=FP8), lambda t: z(4, 16, 256, dtype=FP8), lambda t: t[0],
                lambda t: z(4, 32, 512, dtype=FP8)[:, ::2]],
           at + 1: [lambda t: t.bfloat16(), lambda t: t[:3], lambda t: t[:, :8].contiguous(), lambda t: t.flatten(), lambda t: z(16, 4).t()],
           at + 2: [lambda t: t.float(), lambda t: t[:3], lambda t: z(4, 16, 32, dtype=t.dtype), lambda t: t[:, :8].contiguous(), lambda t: z(4, 16, 128, dtype=t.dtype)[..., ::2]],
           at + 3: [lambda t: t.long(), lambda t: t[:1], lambda t: t[:, :0], lambda t: z(2, 6, dtype=t.dtype)[:, ::2], lambda t: t[0]]}
    for i in ints:
        bad[i] = [lambda t: t.long(), lambda t: t[:1], lambda t: z(4, dtype=t.dtype)[::2], lambda t: t[:, None]]
    if name == "mla_latent_paged":
        bad[0] = [lambda t: t.float(), lambda t: t[..., :-1].contiguous(), lambda t: t[0], lambda t: z(2, 6, 704, dtype=t.dtype)[:, ::2]]
        bad[1] = [lambda t: t.float(), lambda t: t[:64], lambda t: z(256, dtype=t.dtype)[::2], lambda t: None, lambda t: t[:0]]
        bad[2] = [lambda t: t.float(), lambda t: t[:511]]
        bad[3] = [lambda t: t.conj(), lambda t: t[:1], lambda t: t[:, :2].contiguous(), lambda t: t[0], lambda t: t[..., :16].contiguous()]
    if name == "mla_cache_read":
        bad[5] = [lambda t: -1, lambda t: 1 << 23]
    if name == "mla_cache_keep":
        bad[5] = [lambda t: t.long(), lambda t: t[:1], lambda t: z(2, 65, dtype=t.dtype), lambda t: t[0], lambda t: z(2, 10, dtype=t.dtype)[:, ::2]]
    if name.startswith("mla_decode_paged"):
        bad[0] = [lambda t: t.float(), lambda t: t[0], lambda t: z(2, 3, 8, 192, dtype=t.dtype)[:, :, ::2], lambda t: z(2, 3, 4, 128, dtype=t.dtype),
                  lambda t: z(2, 65, 4, 192, dtype=t.dtype), lambda t: t[:, :, :3].contiguous()]
        bad[1] = [lambda t: t.conj(), lambda t: t[:1], lambda t: t[:, :2].contiguous(), lambda t: t[0]]
        bad[8] = [lambda t: t.int(), lambda t: t[:1], lambda t: t[:, :2].contiguous(), lambda t: z(2, 6, dtype=t.dtype)[:, ::2], lambda t: t[0]]
        bad[9] = [lambda t: t.bfloat16(), lambda t: t[:1020], lambda t: t[:, :256].contiguous(), lambda t: z(1024, 1024, dtype=t.dtype)[:, ::2]]
        bad[10] = [lambda t: t[:7], lambda t: t[:, :3].contiguous(), lambda t: t.bfloat16(), lambda t: t.flatten(), lambda t: z(4, 8).t()]
        bad[11] = [lambda t: 0, lambda t: -1, lambda t: 49, lambda t: 1 << 23, lambda t: 2 ** 63 - 1]
        bad[12] = [lambda t: 0.0, lambda t: -1.0, lambda t: float("nan"), lambda t: float("inf"), lambda t: 1e-40]
    for i, changes in bad.items():
        for change in changes:
            args = _args(name)
            args[i] = change(args[i])
            with pytest.raises(RuntimeError, match=name + r"[^:]*: (?!tensors|all tensors)"):
                _gpu_body(name, *args)


@pytest.mark.parametrize("name", OPERATORS)
def test_shapes_without_a_device(name):
    args = [t.to("meta") if isinstance(t, torch.Tensor) else t for t in _args(name)]
    got = getattr(torch.ops.dsv3fp8, name)(*args)
    shapes = {"mla_latent_paged": [(2, 3, 128), (2, 3, 1)], "mla_cache_read": [(2, 20, 512), (2, 20, 64)], "mla_cache_keep": [], "mla_decode_paged": [(2, 3, 512)], "mla_decode_paged_quant": [(2, 3, 512), (2, 3, 4)]}[name]
    got = (got,) if isinstance(got, torch.Tensor) else got
    assert [tuple(t.shape) for t in got or ()] == shapes


def _e4m3(x):
    """The nearest e4m3 values, ties to even."""
    return x.float().to(FP8).double()


def _spread(g, octaves):
    """Rows of 32 values over so many powers of two below the largest, which is any of its binade; every eighth next to a tie of three or seven bits."""
    v = torch.exp2(-octaves * torch.rand(40000, 32, generator=g, dtype=torch.float64)) * (1 + torch.rand(40000, 1, generator=g, dtype=torch.float64))
    mantissa, exponent = torch.frexp(v)
    tie = torch.ldexp((mantissa * 16).round() / 16 + 2.0 ** -5 + 2.0 ** -20 * torch.randn(v.shape, generator=g), exponent)
    v[:, 1::8] = tie[:, 1::8]
    v[:, 0] = v.amax(-1)
    return v.float().double()


def test_two_codes_a_value():
    """What the comment at split_codes (csrc/common.hpp) states of it: off by 2^-9 of the value down to 2^-12 of the largest that shares the scale, by 2^-21 of
    that below; and no better limits hold."""
    v = _spread(torch.Generator().manual_seed(1), 26)
    largest = v.amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(largest)) - 7)                # the largest becomes 128 .. 256
    first = _e4m3(v / scale) * scale
    second = _e4m3((v - first) / (scale / 16)) * (scale / 16)
    error, ratio = (v - first - second).abs(), v / largest
    assert (error <= torch.where(ratio >= 2.0 ** -12, 2.0 ** -9 * v, 2.0 ** -21 * largest)).all()
    assert ((error > 2.0 ** -9 * v) & (ratio > 2.0 ** -13.1)).any() and (error > 2.0 ** -22 * largest)[ratio < 2.0 ** -13].any()


def test_one_code_an_element():
    """What the head of csrc/mla_paged.hip states of a row: off by a sixteenth of the element down to 2^-13.8 of the row's largest (2^-6 of 224 scales), by 2^-10
    of a scale below."""
    v = _spread(torch.Generator().manual_seed(2), 20)
    largest = v.amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(largest / 448)))
    error, limit = (v - _e4m3(v / scale) * scale).abs(), 2.0 ** -6 / 224
    assert (error <= torch.where(v >= limit * largest, v / 16, 2.0 ** -10 * scale)).all()
    assert ((error > v / 16) & (v > 2.0 ** -14.2 * largest)).any()


# a launch has fewer than 2^32 work-items: a workgroup of 320 a row with a query latent, 256 for four rows without one and for 32 positions read back
def test_sizes_that_no_launch_holds(L):
    def write(b, rows, qr):
        return L.lib.dsv3_mla_latent_paged(A16, 2112, A16, A16, A16, _cache(L), A16, A16, A16, A16, b, rows, qr, 512, 64, 1e-6, 1e-6, None)

    def read(b, positions):
        return L.lib.dsv3_mla_cache_read(_cache(L), A16, A16, A16, b, positions, None)
    for rows in (13421773 // 3 + 1, 0x7fffff):
        assert write(3, rows, 1536) == 2
    assert write(9, 67108863 // 9 + 1, 0) == 2 and write(255, 0x7fffff, 0) == 2
    assert read(65, 0x7fffff) == 2 and read(65535, 8193) == 2
