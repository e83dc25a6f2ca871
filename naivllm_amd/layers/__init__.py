from naivllm_amd.layers.attention import Attention, paged_attention_verify, store_kvcache
from naivllm_amd.layers.pages import CachePages

__all__ = ["Attention", "CachePages", "paged_attention_verify", "store_kvcache"]
