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
from .router import NormedRows as NormedRows
from .router import rms_norm as rms_norm
from .router import rms_norm_backward as rms_norm_backward
from .router import rms_norm_workspace as rms_norm_workspace
from .router import route_tokens as route_tokens
from .router import route_tokens_backward as route_tokens_backward
from .router import router_logits as router_logits
from .router import router_logits_backward as router_logits_backward
from .router import router_workspace as router_workspace
