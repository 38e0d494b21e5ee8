"""MI355X-native attention hot path of dl_templates: tiled 2D sliding-window flash attention,
fused 2D rotary encoding and flash attention with separate qk / vo head dims.

Modules mirror the reference's ``src/`` files: ``tiled_swa``, ``fused_rope2d``, ``rope2d``,
``flash_attn``.  For long sequences and serving: ``rope_axes`` (rotation by positions with several axes),
``window_attn`` (attention over a 1D window with sinks, grouped heads), ``paged_cache`` (keys and values in
pages: append and attention), ``paged_cache8`` (the same in 8 bits) and ``page_pool`` (pages handed to
requests).  All device work is done by hand-written gfx950 HIP kernels in ``libdlt_hip.so`` (C ABI in
``include/dlt.h``)."""
__all__ = ["tiled_swa", "fused_rope2d", "rope2d", "flash_attn", "rope_axes", "window_attn", "paged_cache", "paged_cache8", "page_pool"]
