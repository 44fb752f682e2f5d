"""Projections of the HF Llama / Qwen2 models in 8-bit integers (no counterpart in the reference)."""
from __future__ import annotations

from torch import nn

from tilemix_b200.linear.int8_linear import Int8Linear

__all__ = ["quantize_projections_int8"]

_PROJECTIONS = (("self_attn", ("q_proj", "k_proj", "v_proj", "o_proj")), ("mlp", ("gate_proj", "up_proj", "down_proj")))


def quantize_projections_int8(model):
    """Replace the seven projections of every decoder layer by :class:`Int8Linear` (weights in 8 bits with
    a scale for each output feature, activations quantised by token), in place. fp16 or bf16 models,
    plain, TileMix-injected or prepared for prefill (injection and ``prepare_llama_prefill`` come first:
    they want fp16 weights); embeddings, norms and the LM head stay as they are. Returns the model."""
    root = model.model if hasattr(model, "model") else model
    found = []
    for layer in root.layers:
        for part, names in _PROJECTIONS:
            owner = getattr(layer, part)
            for name in names:
                linear = getattr(owner, name)
                if not isinstance(linear, nn.Linear):
                    raise ValueError(f"{part}.{name} is a {type(linear).__name__}, expected an nn.Linear (quantised "
                                     "already, or sharded for tensor parallelism)")
                if not linear.weight.is_cuda:
                    raise RuntimeError("the projections are quantised by a CUDA kernel; move the model to the GPU first")
                found.append((owner, name, linear))
    for owner, name, linear in found:
        setattr(owner, name, Int8Linear(linear))
    return model
