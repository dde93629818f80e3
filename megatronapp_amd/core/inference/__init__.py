
from .dynamic_engine import (DynamicInferenceEngine,
                             get_dynamic_inference_engine)
from .paged_attention import SharedPrefix, paged_attention
from .paged_context import PagedInferenceContext
from .paged_kv_cache import PagedKVCache
