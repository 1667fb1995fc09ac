"""MI355X (gfx950) implementation of the PLM round's dense-linear hot path.

* ``fast_gemm``   — drop-in for the reference's ``plm.fast_gemm`` (``install``, ``fast_gemm``,
                    ``hip_linear``, ``CONFIGS``, ``HALF_DTYPES``).
* ``gemm_tables`` — drop-in for ``plm.gemm_tables`` (``model_shapes``, ``load_table``, ``install``).
* ``verify``      — the fused LM-head verify step (softmax / argmax / nucleus membership).
* ``attention``   — the paged cache of keys and values, its append with the rotation, attention over it.
* ``fp8``         — the linears in 8 bits with a scale per block of 128, and the norm between them.
* ``workloads``   — the measured shapes and their seeded inputs.

All compute runs in ``libplm_amd.so`` (hand-written HIP kernels, C ABI in ``include/plm_amd.h``).
"""

from . import attention, fast_gemm, fp8, gated_lora, gemm_tables, verify, workloads  # noqa: F401
from ._lib import LIBRARY, lib  # noqa: F401
