"""fa2: FlashAttention-2 forward for AMD MI355X (gfx950). The entry point is fa2.kernel.attention.

Serving operators beside it: fa2.packed.attention_packed (sequences of different lengths in one call), fa2.paged
(a K/V cache in pages, in 16 or 8 bits: cache_write, cache_read, attention_paged; windows with sinks, prefixes that a batch
shares), fa2.rotary (positions of one axis or several, heads normalised before) and fa2.pages (a step's pages, on the GPU)."""
