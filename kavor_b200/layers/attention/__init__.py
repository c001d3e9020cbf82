from kavor_b200.layers.attention.paged_attention import (Attention, build_tree_mask, load_kvcache_fp8, store_kvcache,
                                                         store_kvcache_fp8, tree_attention)

__all__ = ["Attention", "build_tree_mask", "load_kvcache_fp8", "store_kvcache", "store_kvcache_fp8",
           "tree_attention"]
