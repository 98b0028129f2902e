"""B200-native fused vector-quantised attention (the hot path of LouChao98/vqtree).

``vqtree_b200.native``  ctypes binding of the C ABI in ``include/vqattn.h`` (libvqattn.so).
``vqtree_b200.api``     tensor-level entry points (assign, aggregates, prefill, decode, paged append / read / attention).
``vqtree_b200.mini_vq``, ``fused_vq_attn``, ``fused_local_attn_rerope``, ``attn_vq``
                        mirrors of the reference's call signatures for this path.
``vqtree_b200.paged_cache``
                        a serving cache: sequences of different lengths in pages of 16 or 8 bits.
"""
__all__ = ["native", "api"]
