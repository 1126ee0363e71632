"""Learner ops: torch oracles (``ref``), kernel bindings (``hip``) and tensor-level
front-ends (``fused``, 8-bit serving: ``int8``)."""
from . import ref  # noqa: F401
from .fused import (DeviceOUNoise, d4pg_critic_loss, expected_q, l2_project, linear, mlp3_forward,  # noqa: F401
                    nstep_assemble, polyak_)
from .int8 import (add_rms_norm_int8, dequantize_rows, linear_int8, mlp3_int8, quantize_rows)  # noqa: F401
