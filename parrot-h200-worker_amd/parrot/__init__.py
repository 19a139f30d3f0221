"""Parrot XL with an MI355X (gfx950) HIP inference path for its MoE layers."""
from .model import GenerationState, ModelConfig, ModelOutput, Parrot
from .paged import PagedBatch, PagedKVCache

__all__ = ["GenerationState", "ModelConfig", "ModelOutput", "PagedBatch", "PagedKVCache", "Parrot"]
