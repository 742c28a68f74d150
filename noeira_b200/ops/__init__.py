from .beam import beam_reorder, beam_select  # noqa: F401
from .gemm import gemm  # noqa: F401
from .kvcache import PagedKVCache, paged_attention, plan_tokens  # noqa: F401
from .status import check_status, device_status  # noqa: F401
