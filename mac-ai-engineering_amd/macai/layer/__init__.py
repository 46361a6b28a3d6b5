"""Parts of the Qwen3.5 / Qwen3-Next decoder layers around the gated delta rule, on MI355X.

The linear-attention layers' producers: the convolution path (q, k, v from the input projection) and the gates (beta, g).
The reference's macai.layer holds the whole decoder layer; only these two parts feed the rule (reference layer/_conv.py,
layer/_gates.py).

The attention layers between them, which the reference leaves to PyTorch: rotary positions, and for serving a paged cache
held in 4 bits with the step's plan, the append and the attention over it."""
from ._conv import ConvQKV, conv_qkv
from ._gates import Gates, gates
from ._kv4 import kv4_append, kv4_attention, kv4_cache, kv4_plan, kv4_read
from ._rotary import Rotary, rotary, rotary_table

__all__ = ["ConvQKV", "conv_qkv", "Gates", "gates", "Rotary", "rotary", "rotary_table", "kv4_append", "kv4_attention",
           "kv4_cache", "kv4_plan", "kv4_read"]
