"""Refusals of the operators with 4-bit weights, their packing and their oracle (CPU
only: every argument is checked on the host before any launch)."""

import ctypes

import pytest
import torch

import kadllm
from kadllm_amd import _lib, layers
from kadllm_amd.ops import (QuantizedWeight, dequantize_weight, quantize_weight,
                            quantized_gated_ffn, quantized_linear)
from oracle import quantized_ref as ref

U8, BF = torch.uint8, torch.bfloat16


def _weight(N=5, K=40, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes, exps = ref.quantize(torch.randn(N, K, generator=g))
    return QuantizedWeight.pack(*ref.parts(codes, exps), cols=K)


def test_names_are_public():
    for name in ("QuantizedWeight", "quantize_weight", "dequantize_weight", "quantized_linear",
                 "quantized_gated_ffn"):
        assert getattr(kadllm, name) is getattr(kadllm.ops, name)
        assert name in kadllm.__all__


def test_oracle_rounds_to_even_and_saturates():
    w = torch.tensor([[7.0, 5.0, 2.5, 1.75, 1.25, 0.75, 0.25, -3.5, 0.2500001, -5.1]])
    codes, exps = ref.quantize(w)
    assert exps.tolist() == [[0]]
    assert ref.dense(codes, exps).tolist() == [[6, 4, 2, 2, 1, 1, 0, -4, 0.5, -6]]
    assert ref.quantize(torch.tensor([[7.001]]))[1].tolist() == [[1]]
    assert ref.quantize(torch.zeros(1, 3))[1].tolist() == [[0]]
    assert ref.quantize(torch.full((1, 3), 1e-40))[1].tolist() == [[-100]]
    assert ref.quantize(torch.tensor([[3e38]]))[1].tolist() == [[125]]
    assert ref.dense(*ref.quantize(torch.tensor([[1.0, float("inf")]]))).isnan().all()


@pytest.mark.parametrize("N, K", [(1, 1), (16, 128), (17, 129), (5, 700), (40, 31), (33, 1024)])
def test_pack_and_unpack(N, K):
    g = torch.Generator().manual_seed(N + K)
    codes = torch.randint(0, 256, (N, -(-K // 2)), generator=g).to(U8)
    scales = torch.randint(27, 253, (N, -(-K // 32)), generator=g).to(U8)
    if K % 2:
        codes[:, -1] &= 15
    w = QuantizedWeight.pack(codes, scales.view(torch.float8_e8m0fnu), cols=K)
    assert (w.rows, w.cols) == (N, K)
    assert w.codes.shape == (-(-N // 16), -(-K // 128), 64, 16)
    assert w.scales.shape == (-(-N // 16), -(-K // 128), 16, 4)
    back = w.unpack()
    assert torch.equal(back[0], codes)
    assert torch.equal(back[1].view(U8), scales)
    # word j of entry l of a block: row l % 16, columns 32 j + 8 (l // 16) to + 7
    for n, k in {(0, 0), (N - 1, K - 1), (N // 2, K // 2), (N // 3, K - 1)}:
        lane, j = n % 16 + 16 * (k % 32 // 8), k % 128 // 32
        byte = int(w.codes[n // 16, k // 128, lane, 4 * j + k % 8 // 2])
        assert byte >> 4 * (k % 2) & 15 == int(codes[n, k // 2]) >> 4 * (k % 2) & 15
        assert int(w.scales.view(U8)[n // 16, k // 128, n % 16, j]) == int(scales[n, k // 32])
    # nothing but zeros past the weight's rows and columns
    assert int((w.codes != 0).sum()) <= int((codes != 0).sum())


def test_pack_takes_torch_types():
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (4, 32), generator=g).to(U8)
    scales = torch.full((4, 2), 120, dtype=U8)
    a = QuantizedWeight.pack(codes, scales)
    b = QuantizedWeight.pack(codes.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e8m0fnu))
    assert a.cols == b.cols == 64 and torch.equal(a.codes, b.codes)


@pytest.mark.parametrize("change, error", [
    (dict(codes=torch.zeros(4, 32)), TypeError),
    (dict(scales=torch.zeros(4, 2)), TypeError),
    (dict(codes=torch.zeros(4, dtype=U8)), ValueError),
    (dict(codes=torch.zeros(4, 0, dtype=U8), scales=torch.zeros(4, 0, dtype=U8)), ValueError),
    (dict(codes=torch.zeros(0, 32, dtype=U8), scales=torch.zeros(0, 2, dtype=U8)), ValueError),
    (dict(scales=torch.full((4, 3), 120, dtype=U8)), ValueError),
    (dict(scales=torch.full((3, 2), 120, dtype=U8)), ValueError),
    (dict(cols=62), ValueError),
    (dict(cols=65), ValueError),
    (dict(cols=64.0), ValueError),
    (dict(scales=torch.full((4, 2), 26, dtype=U8)), ValueError),
    (dict(scales=torch.full((4, 2), 253, dtype=U8)), ValueError),
])
def test_pack_refusals(change, error):
    args = dict(codes=torch.zeros(4, 32, dtype=U8), scales=torch.full((4, 2), 120, dtype=U8))
    args.update(change)
    with pytest.raises(error):
        QuantizedWeight.pack(args.pop("codes"), args.pop("scales"), **args)


@pytest.mark.parametrize("w, error", [
    (torch.zeros(4), ValueError),
    (torch.zeros(4, 0), ValueError),
    (torch.zeros(0, 4), ValueError),
    (torch.zeros(4, 4, dtype=torch.float64), TypeError),
    (torch.zeros(4, 4, dtype=torch.int32), TypeError),
    (torch.zeros(1, 1, dtype=BF).expand(1, 2**20 + 1), ValueError),
    (torch.zeros(4, 4).requires_grad_(), RuntimeError),
    (torch.zeros(4, 4), RuntimeError),  # well-formed, but not on a ROCm device
])
def test_quantize_refusals(w, error):
    with pytest.raises(error):
        quantize_weight(w)


@pytest.mark.parametrize("change, error", [
    (dict(codes=torch.zeros(1, 1, 64, 16)), TypeError),
    (dict(scales=torch.zeros(1, 1, 16, 4, dtype=U8)), TypeError),
    (dict(rows=17), ValueError),
    (dict(rows=0), ValueError),
    (dict(cols=129), ValueError),
    (dict(cols=True), ValueError),
    (dict(codes=torch.zeros(1, 0, 64, 16, dtype=U8)), ValueError),
    (dict(codes=torch.zeros(1, 1, 16, 64, dtype=U8).transpose(2, 3)), ValueError),
])
def test_weight_refusals(change, error):
    w = _weight()
    parts = dict(codes=w.codes, scales=w.scales, rows=w.rows, cols=w.cols)
    QuantizedWeight(**parts)
    with pytest.raises(error):
        QuantizedWeight(**{**parts, **change})


def test_a_weight_is_not_changed():
    w = _weight()
    for name in ("codes", "rows", "other"):
        with pytest.raises(AttributeError):
            setattr(w, name, 3)
    assert "5 x 40" in repr(w)
    import copy
    other = copy.deepcopy(w)
    assert torch.equal(other.codes, w.codes) and other.codes.data_ptr() != w.codes.data_ptr()
    assert w.to("cpu").cols == 40


def test_operators_take_only_weights():
    w, x = _weight(), torch.zeros(3, 40, dtype=BF)
    for bad in ((w.codes, w.scales, 5, 40), w.codes, None):
        with pytest.raises(TypeError):
            dequantize_weight(bad)
        with pytest.raises(TypeError):
            quantized_linear(x, bad)
        for args in ((bad, w, w), (w, bad, w), (w, w, bad)):
            with pytest.raises(TypeError):
                quantized_gated_ffn(x, *args)
    with pytest.raises(RuntimeError):  # well-formed, but not on a ROCm device
        dequantize_weight(w)


def test_dequantize_refuses_types():
    with pytest.raises(TypeError):
        dequantize_weight(_weight(), torch.float64)


@pytest.mark.parametrize("change, error", [
    (dict(x=torch.zeros(3, 41, dtype=BF)), ValueError),
    (dict(x=torch.zeros((), dtype=BF)), ValueError),
    (dict(x=torch.zeros(0, 40, dtype=BF)), ValueError),
    (dict(x=torch.zeros(3, 40, dtype=torch.float64)), TypeError),
    (dict(x=torch.zeros(3, 40, dtype=torch.int32)), TypeError),
    (dict(residual=True), ValueError),
    (dict(residual=torch.float16), ValueError),
    (dict(x=torch.zeros(3, 40, dtype=BF).requires_grad_()), RuntimeError),
    (dict(x=torch.zeros(1, 1, dtype=BF).expand(2**24 + 1, 40)), ValueError),
    (dict(), RuntimeError),  # well-formed, but not on a ROCm device
])
def test_product_refusals(change, error):
    gate, up, down = _weight(), _weight(seed=1), _weight(40, 5)
    x = change.get("x", torch.zeros(3, 40, dtype=BF))
    for call, args, cols in ((quantized_linear, (gate,), 5),
                             (quantized_gated_ffn, (gate, up, down), 40)):
        r = change.get("residual")
        if r is True:
            r = torch.zeros(3, cols + 1, dtype=BF)
        elif r is not None:
            r = torch.zeros(3, cols, dtype=r)
        with pytest.raises(error):
            call(x, *args, residual=r)


def test_ffn_refuses_unlike_shapes():
    x = torch.zeros(3, 40, dtype=BF)
    for args in ((_weight(), _weight(6), _weight(40, 5)), (_weight(), _weight(), _weight(40, 6)),
                 (_weight(), _weight(), _weight(5, 40))):
        with pytest.raises(ValueError):
            quantized_gated_ffn(x, *args)


# the C entry points check by themselves (no launch is reached: no pointer is read)
P = 1 << 20  # an aligned address


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def test_c_quantize_refusals():
    good = dict(w=P, ld=64, dtype=0, codes=P, scales=P, N=3, K=64)
    for change in (dict(w=None), dict(codes=None), dict(scales=None), dict(ld=63), dict(N=0),
                   dict(K=0), dict(K=2**20 + 1, ld=2**21), dict(codes=P + 8),
                   dict(N=2**31 - 1, K=2**20, ld=2**20), dict(dtype=3)):
        a = {**good, **change}
        assert _rc("kad_quantize_weight", a["w"], a["ld"], a["dtype"], a["codes"], a["scales"],
                   a["N"], a["K"], None) < 0, change
        assert _rc("kad_dequantize_weight", a["codes"], a["scales"], a["w"], a["ld"], a["dtype"],
                   a["N"], a["K"], None) < 0, change


def test_a_swiglu_product_takes_no_4_bit_weight():
    x = torch.zeros(2, 40, dtype=BF)
    with pytest.raises(ValueError):
        layers.gemm(x, _weight(), epilogue=layers.EPI_SWIGLU)


def test_c_product_of_as_many_rows_as_a_grid_takes():
    bytes = ctypes.c_int64(0)
    # 2^28 - 1 pieces of 128 columns: 16 of them a workgroup, 2^24 workgroups of 256
    M, K = 617093, 435 * 128
    args = (3, K + 3, 0, M, 20000, K - 3)
    assert _rc("kad_quantized_linear_workspace_bytes", *args, ctypes.byref(bytes)) < 0
    args = (3, K + 3, 0, M - 1, 20000, K - 3)
    assert _rc("kad_quantized_linear_workspace_bytes", *args, ctypes.byref(bytes)) == 0
    assert bytes.value == (M - 1) * K * 2


def test_c_product_refusals():
    n = ctypes.c_int64(0)
    good = dict(x=P, ldx=64, dtype=1, codes=P, scales=P, r=None, ldr=0, y=P, ldy=32, ws=P,
                bytes=1 << 30, M=3, N=32, K=64)
    many = dict(M=3000, N=20000, ldy=20000, K=60)  # rows that are padded first
    assert _rc("kad_quantized_linear_workspace_bytes", P, 64, 1, 3000, 20000, 60,
               ctypes.byref(n)) == 0 and n.value == 3000 * 256
    for change in (dict(x=None), dict(codes=None), dict(scales=None), dict(y=None), dict(ldx=63),
                   dict(ldy=31), dict(r=P, ldr=31), dict(many, ws=None), dict(many, ws=P + 8),
                   dict(many, bytes=10), dict(M=0), dict(M=16 * 65535 + 1), dict(N=0), dict(K=0),
                   dict(N=2**26 + 1, ldy=2**27), dict(dtype=7), dict(codes=P + 4),
                   dict(K=2**20 + 1, ldx=2**21)):
        a = {**good, **change}
        assert _rc("kad_quantized_linear", a["x"], a["ldx"], a["dtype"], a["codes"], a["scales"],
                   a["r"], a["ldr"], a["y"], a["ldy"], a["ws"], a["bytes"], a["M"], a["N"], a["K"],
                   None) < 0, change
    assert _rc("kad_quantized_linear_workspace_bytes", P, 64, 0, 3, 32, 64, None) < 0
    assert _rc("kad_quantized_linear_workspace_bytes", P, 2**20, 2, 2**16, 1, 2**20,
               ctypes.byref(n)) < 0
    assert _rc("kad_quantized_gated_ffn_workspace_bytes", P, 64, 0, 3, 32, 64, None) < 0
    assert _rc("kad_quantized_gated_ffn_workspace_bytes", P, 64, 0, 3, 64, 100,
               ctypes.byref(n)) == 0 and n.value > 0
    ffn = dict(x=P, ldx=64, dtype=0, g=P, gs=P, u=P, us=P, d=P, ds=P, r=None, ldr=0, y=P, ldy=64,
               ws=P, bytes=1 << 30, M=3, H=64, F=100)
    for change in (dict(x=None), dict(g=None), dict(us=None), dict(ds=None), dict(d=P + 8),
                   dict(y=None), dict(ldx=60), dict(ldy=60), dict(r=P, ldr=1), dict(ws=None),
                   dict(bytes=0), dict(M=-1), dict(H=0), dict(F=2**20 + 1), dict(dtype=-1)):
        a = {**ffn, **change}
        assert _rc("kad_quantized_gated_ffn", *list(a.values()), None) < 0, change
