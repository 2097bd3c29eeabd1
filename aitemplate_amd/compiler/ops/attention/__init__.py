from .mem_eff_attention import mem_eff_attention  # noqa: F401
from .paged_attention import paged_kv_append, prefix_attention  # noqa: F401
from .rotary_embedding import rotary_embedding  # noqa: F401
