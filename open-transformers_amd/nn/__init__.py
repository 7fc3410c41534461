"""Neural-network operators of the ROCm backend (mirrors ``repop.nn``)."""

from . import embedding, flash_attention, functional, layer, loss, masked_attention

__all__ = ["embedding", "flash_attention", "functional", "layer", "loss", "masked_attention"]
