"""artlite_amd: artlite's mixture-of-experts FFN layer over GGUF-quantized experts, native to MI355X (gfx950).

The Python API of the reference's MoE operator (``artlite.moe``: ``plan.route``, ``plan.Plan``, ``route.top_k`` /
``deal`` / ``route`` / ``item_weights``), its GGUF row dequantization (``gguf_model``) and a device-resident layer
(``moe.layer.MoELayer``); beside it a model's dense products over 4-bit blocks on device memory (``linear.QLinear``:
projections, output heads; ``ffn.GatedFFN``: the dense feed-forward blocks, forward and backward). All backed by the HIP
library ``libartlite_moe.so`` through ctypes. No torch.
"""

from ._hip import Error, device_count

__all__ = ["Error", "device_count"]
__version__ = "0.1.0"
