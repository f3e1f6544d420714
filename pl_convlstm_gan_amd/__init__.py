"""MI355X-native ConvLSTM rollout engine behind the reference's model interface.

csrc/      hand-written HIP kernels (gfx950) + the C ABI (include/plconvlstm.h)
_lib.py    ctypes binding of libplconvlstm.so
ops.py     pointer/stream plumbing
layers.py  gated linear recurrence, group norm with an activation, counter-based dropout
models.py  ConvLSTMCell / Generator with the reference's signatures and state_dict keys
"""
from .layers import (CounterDropout, GroupNormAct, counter_dropout, gated_linear_scan, gated_linear_step,  # noqa: F401
                     group_norm_act)
from .models import (ConvLSTMCell, DEMAttention, Generator, LUAttention, UpsampleBlock,  # noqa: F401
                     add_coord_channels)

__all__ = ["ConvLSTMCell", "DEMAttention", "Generator", "LUAttention", "UpsampleBlock", "add_coord_channels",
           "CounterDropout", "GroupNormAct", "counter_dropout", "gated_linear_scan", "gated_linear_step", "group_norm_act"]
