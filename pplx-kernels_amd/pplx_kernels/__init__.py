"""MI355X-native MoE dispatch / combine with the ``pplx_kernels`` Python surface
(reference ``src/pplx_kernels/__init__.py:1-16``, minus the NVSHMEM helpers: this build has
no SHMEM layer)."""

from . import ops as ops
from .all_to_all import AllToAll as AllToAll
from .experts import SortedTokens as SortedTokens
from .experts import int8_matmul as int8_matmul
from .experts import quantize_rows as quantize_rows
from .experts import sort_tokens as sort_tokens
from .experts import sort_tokens_backward as sort_tokens_backward
from .experts import unsort_tokens as unsort_tokens
from .experts import unsort_tokens_backward as unsort_tokens_backward
from .loopback import BoundStep as BoundStep
from .loopback import Graph as Graph
from .loopback import LoopbackWorld as LoopbackWorld
