"""fa2: FlashAttention-2 forward for AMD MI355X (gfx950). The entry point is fa2.kernel.attention.

Serving operators beside it: fa2.packed.attention_packed (sequences of different lengths in one call), fa2.paged
(a K/V cache in pages, in 16 or 8 bits: cache_write, cache_read, attention_paged) and fa2.rotary (positions)."""
