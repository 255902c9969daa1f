"""``kadllm.ops`` (src/kadllm/ops.py) on the HIP path: kadllm_amd.ops, including
the validation helpers the reference's benchmark imports (``_gdn_launch``,
benchmarks/grbeam.py:99)."""

from kadllm_amd.ops import (PrefixBlocks, QuantizedWeight, _backend, _gdn_launch,  # noqa: F401
                            _same_device, _width, block_prefix_attention, causal_conv1d,
                            dequantize_weight, gated_delta, merge_attention, prefix_attention,
                            prefix_block_tables, quantize_weight, quantized_gated_ffn,
                            quantized_linear, write_prefix_blocks)
