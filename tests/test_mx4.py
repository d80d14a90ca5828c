"""Microscaled 4-bit numbers and pages of 4-bit rows on the host: what is refused, shapes, layers and pools (no kernel runs)."""
import pytest
import torch

FP8, FP4, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
A16 = 0x1000            # an address that is never looked at


@pytest.fixture(scope="module")
def L():
    from dsv3fp8 import _lib
    return _lib


@pytest.mark.parametrize("entry", ["dsv3_mx4_quant", "dsv3_mx4_dequant"])
def test_conversion_validation(L, entry):
    quant = entry == "dsv3_mx4_quant"

    def call(codes=A16, s=A16, wide=A16, dtype=L.BF16, numel=128, last=64):
        f = getattr(L.lib, entry)
        return f(wide, dtype, codes, s, numel, last, None) if quant else f(codes, s, wide, dtype, numel, last, None)
    for name in ("codes", "s", "wide"):
        assert call(**{name: None}) == 1
    assert call(codes=A16 + 2) == 4 and call(wide=A16 + 8) == 4
    assert call(dtype=3) == 5 and call(dtype=-1) == 5
    for bad in (dict(last=48), dict(last=0), dict(numel=-64), dict(last=-64), dict(numel=96), dict(numel=(1 << 37) + 64)):
        assert call(**bad) == 2, bad
    assert call(numel=0, codes=None) == 0 and call(numel=0, last=0, codes=None) == 0


def test_product_validation(L):
    def call(a=A16, a_s=A16, kind=L.MX4, b=A16, b_s=A16, c=A16, dtype=L.BF16, m=4, n=64, k=256, ws=None, wsb=0):
        return L.lib.dsv3_mx4_gemm(a, a_s, kind, b, b_s, c, dtype, m, n, k, ws, wsb, None)
    for name in ("a", "a_s", "b", "b_s", "c"):
        assert call(**{name: None}) == 1
        assert call(**{name: A16 + (2 if name.endswith("_s") else 8)}) == 4
    assert call(k=512, a_s=A16 + 8) == 4 and call(k=1024, b_s=A16 + 4) == 4      # (pieces of 16 bytes are fetched)
    assert call(kind=2) == 5 and call(kind=-1) == 5 and call(dtype=3) == 5
    for bad in (dict(m=-1), dict(n=-1), dict(k=-128), dict(k=64), dict(k=192), dict(k=(1 << 22) + 128), dict(m=1 << 31), dict(n=1 << 31)):
        assert call(**bad) == 2, bad
    assert call(m=0, a=None) == 0 and call(n=0, b=None) == 0
    sizes = dict(m=4096, n=7168, k=7168)
    for kind in (L.MX4, L.E4M3):
        need = L.lib.dsv3_mx4_gemm_workspace_bytes(kind, 4096, 7168, 7168)
        assert need > 0 and L.lib.dsv3_mx4_gemm_workspace_bytes(kind, 1, 7168, 7168) == 0
        assert call(kind=kind, **sizes) == 6 and call(kind=kind, ws=A16, wsb=need - 1, **sizes) == 6 and call(kind=kind, ws=A16 + 16, wsb=need, **sizes) == 6
    assert L.lib.dsv3_mx4_gemm_workspace_bytes(7, 4096, 7168, 7168) == 0 and L.lib.dsv3_mx4_gemm_workspace_bytes(0, 4096, 7168, 100) == 0
    # more tiles than a launch holds: refused before anything is launched
    huge = dict(m=0x7fffff00, n=0x7fffff00, k=128)
    assert call(ws=A16, wsb=1 << 62, **huge) == 2
    assert call(m=1, n=0x7fffff00) == 2


def _gpu_body(name, *args):
    op = getattr(torch.ops.dsv3fp8, name).default
    return op.redispatch(torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA), *args)


def _args(name):
    codes, scales = torch.zeros(6, 128, dtype=torch.uint8).view(FP4), torch.full((6, 8), 127, dtype=torch.uint8).view(E8M0)
    if name == "mx4_quant":
        return [torch.zeros(6, 256, dtype=torch.bfloat16)]
    if name == "mx4_dequant":
        return [codes, scales, 0]
    return [codes.view(torch.uint8)[:4].clone().view(FP4), scales.view(torch.uint8)[:4].clone().view(E8M0), codes, scales, 0]


@pytest.mark.parametrize("name", ["mx4_quant", "mx4_dequant", "mx4_gemm"])
def test_operators_refuse_the_host_and_two_devices(name):
    with pytest.raises(RuntimeError, match="on the GPU"):
        _gpu_body(name, *_args(name))
    with pytest.raises(NotImplementedError):
        getattr(torch.ops.dsv3fp8, name)(*_args(name))
    for at, t in enumerate(_args(name)):
        if isinstance(t, torch.Tensor) and name != "mx4_quant":
            args = _args(name)
            args[at] = t.to("meta")
            with pytest.raises(RuntimeError, match="one device"):
                _gpu_body(name, *args)


def _u8(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("name", ["mx4_quant", "mx4_dequant", "mx4_gemm"])
def test_operators_refuse_what_their_kernels_cannot_read(name):
    strided = lambda t: torch.zeros(t.size(0), 2 * t.size(1), dtype=torch.uint8).view(t.dtype)[:, ::2]  # noqa: E731
    codes = [lambda t: _u8(t), lambda t: t[:, :64].contiguous() if t.dtype == FP8 else _u8(t)[:, :64].contiguous().view(t.dtype), strided, lambda t: t[:3], lambda t: t[0]]
    scales = [lambda t: _u8(t), lambda t: torch.ones(*t.shape), lambda t: _u8(t)[:, :4].contiguous().view(t.dtype), strided, lambda t: t[:3], lambda t: t[0]]
    bad = {"mx4_quant": {0: [lambda t: t[:, :40].contiguous(), lambda t: t[:, ::2], lambda t: t.t(), lambda t: t[0, 0]]}, "mx4_dequant": {0: codes, 1: scales},
           "mx4_gemm": {0: codes[:3] + [lambda t: t[:3], lambda t: t[0]], 1: scales, 2: codes, 3: scales}}[name]
    for i, changes in bad.items():
        for change in changes:
            args = _args(name)
            args[i] = change(args[i])
            with pytest.raises(RuntimeError, match=name + r"[^:]*: (?!tensors|all tensors)"):
                _gpu_body(name, *args)
    if name == "mx4_quant":
        with pytest.raises(TypeError, match="dtype"):
            _gpu_body(name, torch.zeros(2, 32, dtype=torch.float64))
    if name == "mx4_gemm":
        a, a_s, b, b_s, _ = _args(name)
        for x, xs in ((torch.zeros(4, 256, dtype=FP8), torch.ones(4, 1)), (torch.zeros(4, 256, dtype=FP8), torch.ones(4, 2, dtype=torch.bfloat16)),
                      (torch.zeros(4, 512, dtype=FP8)[:, ::2], torch.ones(4, 2)), (torch.zeros(4, 128, dtype=FP8), torch.ones(4, 1)),
                      (torch.zeros(4, 256, dtype=FP8), torch.ones(2, 4).t()), (torch.zeros(4, 256, dtype=torch.bfloat16), torch.ones(4, 2)),
                      (torch.zeros(4, 256, dtype=FP8), torch.ones(3, 2)), (torch.zeros(256, dtype=FP8)[0], torch.ones(1))):
            with pytest.raises(RuntimeError, match="mx4_gemm"):
                _gpu_body(name, x, xs, b, b_s, 0)
        # a last dimension of 32's but not of 128's
        with pytest.raises(RuntimeError, match="multiple of 128"):
            _gpu_body(name, *(_u8(t)[..., :n].contiguous().view(t.dtype) for t, n in ((a, 48), (a_s, 3), (b, 48), (b_s, 3))), 0)


def test_functions_refuse():
    import dsv3fp8
    for x in (torch.zeros(4, 64)[:, ::2], torch.zeros(4, 48)):
        with pytest.raises(AssertionError):
            dsv3fp8.mx4_quant(x)
    a, a_s, b, b_s, _ = _args("mx4_gemm")
    for args in ((a[:, ::2], a_s, b, b_s), (a, a_s, b, b_s[:, ::2])):
        with pytest.raises(AssertionError):
            dsv3fp8.mx4_gemm(*args)
    with pytest.raises(AssertionError):
        dsv3fp8.mx4_dequant(a, a_s[:, ::2])


def test_shapes_without_a_device():
    y, s = torch.ops.dsv3fp8.mx4_quant(torch.zeros(2, 3, 96, device="meta"))
    assert y.shape == (2, 3, 48) and y.dtype == FP4 and s.shape == (2, 3, 3) and s.dtype == E8M0
    assert torch.ops.dsv3fp8.mx4_dequant(y, s, 2).shape == (2, 3, 96) and torch.ops.dsv3fp8.mx4_dequant(y, s, 1).dtype == torch.float16
    b, b_s = torch.empty(7, 64, dtype=FP4, device="meta"), torch.empty(7, 4, dtype=E8M0, device="meta")
    assert torch.ops.dsv3fp8.mx4_gemm(torch.empty(2, 3, 64, dtype=FP4, device="meta"), torch.empty(2, 3, 4, dtype=E8M0, device="meta"), b, b_s, 0).shape == (2, 3, 7)
    assert torch.ops.dsv3fp8.mx4_gemm(torch.empty(5, 128, dtype=FP8, device="meta"), torch.empty(5, 1, device="meta"), b, b_s, 2).dtype == torch.float32


# ---------------------------------------------------------------------------------------------------------- layers

def test_layers_of_4_bit_weights():
    from dsv3fp8 import model
    lin = model.Linear(256, 48, bias=True, dtype=FP4)
    assert lin.weight.shape == (48, 128) and lin.weight.dtype == FP4 and lin.scale.shape == (48, 8) and lin.scale.dtype == E8M0 and lin.weight.scale is lin.scale
    with pytest.raises(ValueError, match="multiple of 128"):
        model.Linear(192, 48, dtype=FP4)
    assert not model._eight_bits(lin.weight) and model._eight_bits(model.Linear(128, 8, dtype=FP8).weight) and not model._eight_bits(model.Linear(128, 8).weight)
    state = {k: v.clone() for k, v in lin.state_dict().items()}
    _u8(state["weight"]).fill_(0x21)
    _u8(state["scale"]).fill_(130)
    lin.load_state_dict(state)
    assert (_u8(lin.weight.data) == 0x21).all() and (_u8(lin.scale.data) == 130).all()


def test_ways_of_linear(monkeypatch):
    """Which operators a 4-bit weight's product consists of."""
    from dsv3fp8 import model
    calls = []
    for name, result in (("mx4_dequant", lambda w, s: torch.zeros(48, 256)), ("act_quant", lambda x, *a: (x, "scales")), ("mx4_quant", lambda x: (x, "bytes")),
                         ("mx4_gemm", lambda a, s, w, ws: torch.zeros(*a.shape[:-1], 48))):
        monkeypatch.setattr(model, name, lambda *a, name=name, result=result: (calls.append((name, a)), result(*a))[1])
    lin, x = model.Linear(256, 48, dtype=FP4), torch.zeros(2, 3, 256)
    monkeypatch.setattr(model, "gemm_impl", "bf16")
    assert lin(x).shape == (2, 3, 48) and [c[0] for c in calls] == ["mx4_dequant"]
    monkeypatch.setattr(model, "gemm_impl", "fp8")
    for kind, first in (("e4m3", "act_quant"), ("mx4", "mx4_quant")):
        calls.clear()
        monkeypatch.setattr(model, "mx4_activations", kind)
        assert lin(x).shape == (2, 3, 48) and [c[0] for c in calls] == [first, "mx4_gemm"]
        assert calls[1][1][2] is lin.weight and calls[1][1][3] is lin.scale
    assert model.linear(x, lin.weight, torch.ones(48)).sum() == 2 * 3 * 48
    monkeypatch.setattr(model, "mx4_activations", "bf16")
    with pytest.raises(ValueError, match="mx4_activations"):
        lin(x)


def test_fused_paths_leave_4_bit_weights_alone(monkeypatch):
    from dsv3fp8 import model
    monkeypatch.setattr(model.Linear, "dtype", FP4)
    monkeypatch.setattr(model, "gemm_impl", "fp8")
    args = model.ModelArgs(dim=256, n_heads=2, q_lora_rank=128, max_batch_size=2, max_seq_len=64, n_routed_experts=4, n_activated_experts=2, n_expert_groups=1, n_limited_groups=1, moe_inter_dim=128)
    mla, mlp, moe = model.MLA(args), model.MLP(256, 128), model.MoE(args)
    x = torch.zeros(1, 2, 256, dtype=torch.bfloat16)
    assert not mla.stack_a() and not mlp.stack_13() and not moe._grouped_ok(x[0]) and mla._latent_kernel_ok(x) is None
    with torch.no_grad():
        assert mla._kernels_ok(x, 0, torch.zeros(2, 32, dtype=torch.complex64)) is None and not mla._paged_ok(x, torch.zeros(1, 2, 32, dtype=torch.complex64))


def test_pools_of_4_bit_rows():
    from dsv3fp8.model import LatentPages
    c = LatentPages(3, 24, bits=4)
    assert c.kv.shape == (3, 24, 256) and c.kv.dtype == FP4 and c.scale.shape == (3, 24, 16) and c.scale.dtype == E8M0
    assert c.pe.shape == (3, 24, 64) and c.pe.dtype == torch.bfloat16 and (_u8(c.kv) == 0).all() and (_u8(c.scale) == 127).all()
    for bits in (2, 16, 0, 5):
        with pytest.raises(ValueError, match="4 and 8"):
            LatentPages(3, 24, bits=bits)
    with pytest.raises(ValueError):
        LatentPages(0, 24, bits=4)


# ----------------------------------------------------------------------------------------------------------- pages

def _cache(L, **change):
    from ctypes import byref
    fields = dict(kv=A16, kv_scale=A16, pe=A16, pages=4, page_size=64, table=A16, table_width=2, kv_bits=4) | change
    return byref(L.MlaPages(**fields))


def test_pages_validation(L):
    def read(**change):
        return L.lib.dsv3_mla_cache_read(_cache(L, **change), A16, A16, A16, 2, 100, None)

    def keep(**change):
        return L.lib.dsv3_mla_cache_keep(_cache(L, **change), A16, A16, A16, 2, 5, None)

    def write(**change):
        return L.lib.dsv3_mla_latent_paged(A16, 2112, A16, A16, A16, _cache(L, **change), A16, A16, A16, A16, 2, 3, 1536, 512, 64, 1e-6, 1e-6, None)

    def attend(**change):
        return L.lib.dsv3_mla_decode_paged(A16, A16, _cache(L, **change), A16, A16, A16, A16, A16, A16, 2, 3, 100, 4, 128, 64, 128, 512, 0.1, A16, 1 << 30, None)
    for call in (read, keep, write, attend):
        for bits in (1, 2, 5, 16, -4):
            assert call(kv_bits=bits) == 5
        assert call(kv_scale=A16 + 4) == 4 and call(kv_scale=A16 + 8) == 4 and call(kv=A16 + 8) == 4      # a row's scales are read at once
        assert call(kv=None) == 1 and call(kv_scale=None) == 1 and call(pages=0) == 2 and call(page_size=12) == 2


def _paged_args(name):
    z = torch.zeros
    i32 = dict(dtype=torch.int32)
    cache = [z(4, 16, 256, dtype=torch.uint8).view(FP4), torch.full((4, 16, 16), 127, dtype=torch.uint8).view(E8M0), z(4, 16, 64, dtype=torch.bfloat16), z(2, 3, **i32)]
    if name == "mla_latent_paged":
        return [z(2, 3, 128 + 576, dtype=torch.bfloat16), z(128, dtype=torch.bfloat16), z(512, dtype=torch.bfloat16), z(2, 3, 32, dtype=torch.complex64), *cache,
                z(2, **i32), z(2, **i32), 1e-6, 1e-6]
    if name == "mla_cache_read":
        return [*cache, z(2, **i32), 20]
    if name == "mla_cache_keep":
        return [*cache, z(2, **i32), z(2, 5, **i32), z(2, **i32)]
    return [z(2, 3, 4, 192, dtype=torch.bfloat16), z(2, 3, 32, dtype=torch.complex64), *cache, z(2, **i32), z(2, **i32), z(2, 3, dtype=torch.int64),
            z(1024, 512, dtype=FP8), z(8, 4), 20, 0.1]


@pytest.mark.parametrize("name,at", [("mla_latent_paged", 4), ("mla_cache_read", 0), ("mla_cache_keep", 0), ("mla_decode_paged", 2), ("mla_decode_paged_quant", 2)])
def test_operators_on_pages_refuse(name, at):
    """Codes of one form with scales of the other, and pools that do not fit."""
    with pytest.raises(RuntimeError, match="on the GPU"):
        _gpu_body(name, *_paged_args(name))
    codes = [lambda t: _u8(t), lambda t: torch.zeros(4, 16, 512, dtype=FP8), lambda t: _u8(t)[..., :128].contiguous().view(FP4), lambda t: t[:3], lambda t: t[0],
             lambda t: torch.zeros(4, 32, 256, dtype=torch.uint8).view(FP4)[:, ::2], lambda t: torch.zeros(4, 16, 512, dtype=torch.uint8).view(FP4)]
    scales = [lambda t: _u8(t), lambda t: torch.ones(4, 16), lambda t: t[:3], lambda t: _u8(t)[..., :8].contiguous().view(E8M0), lambda t: t[:, :8],
              lambda t: torch.zeros(4, 16, 32, dtype=torch.uint8).view(E8M0)[..., ::2]]
    for i, changes in ((at, codes), (at + 1, scales)):
        for change in changes:
            args = _paged_args(name)
            args[i] = change(args[i])
            with pytest.raises(RuntimeError, match=name + r"[^:]*: (?!tensors|all tensors)"):
                _gpu_body(name, *args)


def test_shapes_of_pages_without_a_device():
    args = [t.to("meta") if isinstance(t, torch.Tensor) else t for t in _paged_args("mla_cache_read")]
    kv, pe = torch.ops.dsv3fp8.mla_cache_read(*args)
    assert kv.shape == (2, 20, 512) and kv.dtype == torch.bfloat16 and pe.shape == (2, 20, 64)


# The e4m3 codes that the attention meets a row's codes as: every magnitude times 2^6 .. 2^-8 is one of them
def test_widened_codes_are_e4m3():
    magnitudes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    for step in range(15):
        v = magnitudes * 2.0 ** (6 - step)
        assert torch.equal(v.float().to(FP8).double(), v)
    assert not torch.equal((magnitudes * 2.0 ** -9).float().to(FP8).double(), magnitudes * 2.0 ** -9)


@pytest.mark.parametrize("behind", [0, 4, 7, 8, -1])
def test_what_lies_behind_the_struct_of_pages_is_not_read(L, behind):
    """A host's struct has seven fields, of which page_size alone says that rows are e4m3; what follows it in the host's memory is not the library's."""
    import ctypes

    class Seven(ctypes.Structure):
        _fields_ = [("kv", ctypes.c_void_p), ("kv_scale", ctypes.c_void_p), ("pe", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page_size", ctypes.c_int),
                    ("table", ctypes.c_void_p), ("table_width", ctypes.c_int64)]

    class Held(ctypes.Structure):
        _fields_ = [("pages", Seven), ("behind", ctypes.c_int * 4)]
    # kv_scale: 4-byte aligned, which is what e4m3 rows ask for
    held = Held(Seven(A16, A16 + 4, A16, 4, 64, A16, 2), (ctypes.c_int * 4)(*[behind] * 4))
    cache = ctypes.cast(ctypes.byref(held), ctypes.POINTER(L.MlaPages))
    # (a null pointer is looked for behind the struct's checks, so that nothing is launched)
    assert L.lib.dsv3_mla_cache_read(cache, None, A16, A16, 2, 100, None) == 1
    assert L.lib.dsv3_mla_cache_keep(cache, None, A16, A16, 2, 5, None) == 1
    assert L.lib.dsv3_mla_latent_paged(None, 2112, A16, A16, A16, cache, A16, A16, A16, A16, 2, 3, 1536, 512, 64, 1e-6, 1e-6, None) == 1
    assert L.lib.dsv3_mla_decode_paged(None, A16, cache, A16, A16, A16, A16, A16, A16, 2, 3, 100, 4, 128, 64, 128, 512, 0.1, A16, 1 << 30, None) == 1
    assert L.lib.dsv3_mla_decode_paged_quant(None, A16, cache, A16, A16, A16, A16, A16, A16, A16, 2, 3, 100, 4, 128, 64, 128, 512, 0.1, A16, 1 << 30, None) == 1
    assert ctypes.sizeof(L.MlaPages) == ctypes.sizeof(Seven)


def _moe(monkeypatch):
    from dsv3fp8 import model
    monkeypatch.setattr(model.Linear, "dtype", FP8)
    monkeypatch.setattr(model, "gemm_impl", "fp8")
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    monkeypatch.setattr(torch, "get_default_dtype", lambda: torch.bfloat16)
    try:
        moe = model.MoE(model.ModelArgs(dim=256, n_routed_experts=4, n_activated_experts=2, n_expert_groups=1, n_limited_groups=1, moe_inter_dim=128, n_shared_experts=1))
    finally:
        torch.set_default_dtype(old)
    for module in moe.modules():
        if isinstance(module, model.Linear):
            module.weight.data.view(torch.uint8).fill_(0x38)
            module.scale.data.fill_(1.0)
    return model, moe


@pytest.mark.parametrize("expert,name", [(None, None), (0, "w1"), (0, "w2"), (0, "w3"), (2, "w1"), (3, "w2"), (1, "w3")])
def test_experts_of_which_some_are_of_4_bits(monkeypatch, expert, name):
    """One layer of four bits among the routed experts: they are not grouped, and no weight is moved."""
    from test_mla_dispatch import _OnGpu
    model, moe = _moe(monkeypatch)
    x = torch.zeros(2, 256, dtype=torch.bfloat16).as_subclass(_OnGpu)
    if expert is None:
        assert moe._grouped_ok(x)
        moe.stack_experts()
        assert moe._grouped_ok(x) and moe._shared_stacked and moe._stacked[0].shape == (5, 256, 256)
        return
    lin = getattr(moe.experts[expert], name)
    setattr(moe.experts[expert], name, model.Linear(lin.in_features, lin.out_features, dtype=FP4))
    assert not moe._grouped_ok(x) and moe._stacked is None


@pytest.mark.parametrize("name", ["w1", "w2", "w3"])
def test_a_shared_expert_with_a_layer_of_4_bits(monkeypatch, name):
    """It stays by itself; the routed experts are grouped without it."""
    from test_mla_dispatch import _OnGpu
    model, moe = _moe(monkeypatch)
    sh = moe.shared_experts
    lin = getattr(sh, name)
    setattr(sh, name, type(lin)(lin.in_features, lin.out_features, dtype=FP4))
    before = {n: getattr(sh, n).weight.data_ptr() for n in ("w1", "w2", "w3")}
    assert moe._grouped_ok(torch.zeros(2, 256, dtype=torch.bfloat16).as_subclass(_OnGpu))
    moe.stack_experts()
    assert not moe._shared_stacked and moe._stacked[0].shape == (4, 256, 256) and before == {n: getattr(sh, n).weight.data_ptr() for n in before}


def _four_bit_linear():
    from dsv3fp8 import model
    lin = model.Linear(256, 48, bias=True, dtype=FP4)
    _u8(lin.weight.data).copy_(torch.randint(0, 256, (48, 128)).to(torch.uint8))
    _u8(lin.scale.data).copy_(torch.randint(0, 255, (48, 8)).to(torch.uint8))
    return lin


@pytest.mark.parametrize("convert", ["to", "half", "float", "double", "bfloat16", "in a model", "to a device and type"])
def test_conversions_of_a_layer_leave_its_codes(convert):
    """torch has no conversion of float4_e2m1fn_x2 (an error on the host, a fault on the GPU): codes and scales stay what they are, the bias is converted."""
    lin = _four_bit_linear()
    codes, scale, weight = _u8(lin.weight.data).clone(), _u8(lin.scale.data).clone(), lin.weight
    module = torch.nn.Sequential(torch.nn.LayerNorm(4), lin) if convert == "in a model" else lin
    dtype = {"half": torch.float16, "float": torch.float32, "double": torch.float64}.get(convert, torch.bfloat16)
    if convert in ("to", "in a model"):
        module.to(dtype)
    elif convert == "to a device and type":
        module.to("cpu", dtype)
    else:
        getattr(module, convert)()
    assert lin.weight is weight and lin.weight.scale is lin.scale and lin.weight.dtype == FP4 and lin.scale.dtype == E8M0 and lin.bias.dtype == dtype
    assert torch.equal(_u8(lin.weight.data), codes) and torch.equal(_u8(lin.scale.data), scale)


def test_layers_of_4_bit_weights_on_other_devices():
    lin = _four_bit_linear()
    with pytest.raises(TypeError, match="4 bits"):
        lin.type(torch.float32)
    assert lin.weight.shape == (48, 128) and lin.weight.dtype == FP4
    lin.to("meta")
    assert lin.weight.device.type == "meta" and lin.weight.dtype == FP4 and lin.scale.dtype == E8M0 and lin.weight.shape == (48, 128)
    lin.to_empty(device="cpu")
    assert lin.weight.device.type == "cpu" and lin.weight.dtype == FP4 and lin.scale.shape == (48, 8)
    # e4m3 weights are converted as before
    from dsv3fp8 import model
    assert model.Linear(128, 8, dtype=FP8).to(torch.bfloat16).weight.dtype == torch.bfloat16


def test_layers_without_a_weight_are_moved_as_before():
    from dsv3fp8 import model
    lin = model.Linear(128, 8, bias=True)
    del lin.weight
    assert lin.to(torch.float16).bias.dtype == torch.float16
