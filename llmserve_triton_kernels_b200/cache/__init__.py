from .allocator import IdAllocator, OutOfPages  # noqa: F401
from .manager import CacheManager, CompositeView, PagedKVView, PageGroup, StateView  # noqa: F401


def num_pages_for_budget(cache_specs, page_size: int, element_size: int, budget_bytes: int) -> int:
    """How many pages each group gets when ``budget_bytes`` is shared by all of them
    (src/llmserve/kvcache/paged.py:221-227: bytes of one page = 2 * layers * kv_heads * page_size *
    head_dim * element size).  An element size of 1 is an 8-bit cache's, which keeps a byte more for every head's vector."""
    from ..parts.base import PagedKVSpec, PagedRowSpec, flat_specs

    cache_specs = list(flat_specs(cache_specs))

    per_page = sum(
        2 * s.kv_heads * page_size * (s.head_dim * element_size + (element_size == 1)) for s in cache_specs if isinstance(s, PagedKVSpec)
    ) + sum(s.width * page_size * element_size for s in cache_specs if isinstance(s, PagedRowSpec))
    return max(1, budget_bytes // per_page) if per_page else 1
