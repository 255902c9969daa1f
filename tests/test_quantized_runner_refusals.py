"""What the one-call passes refuse of layers with 4-bit weights (CPU only: they look at
the whole model before the first launch, so no pointer of these is read)."""

import ctypes

import pytest

from kadllm_amd import _lib
from kadllm_amd.native_layers import _Layer, _Model, _PrefillArgs, _Prefix, _StepArgs

P = 1 << 20  # an aligned address
WEIGHTS = ("w_gu", "w_up", "w_down", "w_in", "w_ab", "w_out", "w_qkv", "w_o", "conv_w", "A_log",
           "dt_bias", "norm_w", "q_norm", "k_norm", "input_norm", "post_norm")
SCALES = ("s_gate", "s_up", "s_down", "s_in", "s_out", "s_qkv", "s_o")


def _call(name, model, args, layers):
    """The status of a pass over two good layers, changed by the dicts."""
    structs = (_Layer * 2)()
    for i, layer in enumerate(structs):
        layer.linear = int(i == 0)
        for field in WEIGHTS + SCALES:
            setattr(layer, field, P)
        for field, value in layers.get(i, {}).items():
            setattr(layer, field, value)
    sizes = dict(n_layers=2, hidden=256, ffn=384, conv_dim=768, kd=256, vd=256, gdn_cols=1104,
                 ab_rows=8, k_heads=2, v_heads=2, k_dim=128, v_dim=128, q_heads=2, kv_heads=1,
                 head_dim=128, rot=64, eps=1e-6, gdn_scale=1.0, attn_scale=1.0, inv_freq=P)
    m = _Model(layers=structs, **{**sizes, **model})
    arrays = (ctypes.c_void_p * 2)(P, P)
    pointers = dict(x=P, n=P, h=P, mixed=P, q=P, g=P, beta=P)
    if name == "kad_qwen_prefill":
        a = dict(layers=2, B=1, L=4, fuse_conv=0, state0=ctypes.addressof(arrays),
                 state1=ctypes.addressof(arrays), proj=P, conv=P, chunk_ws=P, **pointers)
        a = _PrefillArgs(**{**a, **args})
    else:
        prefix = (_Prefix * 2)()
        a = dict(B=1, W=4, Wp=4, T=1, keep=0, prefix=ctypes.addressof(prefix), qkv=P, rows_ws=P,
                 k_ws=P, v_ws=P, ab=P, **pointers)
        a = _StepArgs(**{**a, **args})
    rc = getattr(_lib.load(), name)(ctypes.addressof(m), ctypes.addressof(a), None)
    return rc, _lib.load().kad_last_error().decode()


BOTH = ("kad_qwen_prefill", "kad_qwen_decode_step")


@pytest.mark.parametrize("name", BOTH)
@pytest.mark.parametrize("model, args, layers, word", [
    # the widths of the weights' rows
    (dict(hidden=192), {}, {}, "192 columns"),
    (dict(ffn=320), {}, {}, "320 columns"),
    (dict(vd=264), {}, {}, "264 columns"),
    (dict(head_dim=96), {}, {}, "192 columns"),
    (dict(ffn=2**20 + 128), {}, {}, "columns"),
    # the last layer's alone
    (dict(ffn=320), {}, {0: dict(s_gate=None, s_up=None, s_down=None)}, "layer 1"),
    # one of the three of the feed-forward block
    ({}, {}, {1: dict(s_gate=None)}, "layer 1"),
    ({}, {}, {1: dict(s_up=None)}, "layer 1"),
    ({}, {}, {1: dict(s_down=None)}, "layer 1"),
    # alignment and null pointers
    ({}, dict(n=P + 2), {}, "aligned"),
    ({}, dict(h=P + 8), {}, "aligned"),
    ({}, dict(mixed=P + 8), {}, "aligned"),
    ({}, {}, {1: dict(w_qkv=P + 8)}, "aligned"),
    ({}, {}, {1: dict(s_o=P + 4)}, "aligned"),
    ({}, {}, {0: dict(w_in=None)}, "null"),
    ({}, {}, {0: dict(w_up=None)}, "null"),
    # more rows than the products take
    ({}, dict(B=2**16), {}, "outputs"),
])
def test_passes_refuse_before_the_first_launch(name, model, args, layers, word):
    args = dict(args)
    if "B" in args:
        args["L" if name == BOTH[0] else "W"] = 16
    rc, said = _call(name, model, args, layers)
    assert rc == -1 and word in said, (rc, said)


def test_no_convolution_is_fused_into_a_4_bit_projection():
    # (the fused product takes a bf16 weight: four times the bytes of these codes)
    rc, said = _call("kad_qwen_prefill", {}, dict(fuse_conv=1, conv_bytes=1 << 30), {})
    assert rc == -1 and "convolution" in said, (rc, said)
    # (no layer, no launch)
    assert _call("kad_qwen_prefill", {}, dict(fuse_conv=1, layers=0), {})[0] == 0
