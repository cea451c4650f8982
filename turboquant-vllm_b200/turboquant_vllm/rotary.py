"""Frequencies of rotary positions, plain and scaled for long contexts, for :func:`turboquant_vllm.kernels.tq4_rotary`.

Host arithmetic in fp64: a model makes its frequencies once.  ``scaling`` takes the dictionaries that HuggingFace configurations
carry as ``rope_scaling`` / ``rope_parameters``.
"""

from __future__ import annotations

import math
from typing import Any

import torch


def _needed(scaling: dict[str, Any], kind: str, key: str) -> Any:
    value = scaling.get(key)
    if value is None:
        raise ValueError(f"{kind} scaling needs {key}")
    return value


def _yarn(inv_freq: torch.Tensor, dim: int, base: float, scaling: dict[str, Any]) -> tuple[torch.Tensor, float]:
    """Frequencies that turn often over the original context stay, those that turn rarely are divided by the factor, with a ramp
    between the two (Peng et al., "YaRN", section 3); the attention factor is that of their equation 22."""
    factor = float(_needed(scaling, "yarn", "factor"))
    original = float(_needed(scaling, "yarn", "original_max_position_embeddings"))

    def place(turns: float) -> float:  # of the frequency that makes so many turns over the original context
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = place(float(scaling.get("beta_fast") or 32)), place(float(scaling.get("beta_slow") or 1))
    if scaling.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)

    def mscale(m: float) -> float:
        return 1.0 if factor <= 1 else 0.1 * m * math.log(factor) + 1.0

    attention = scaling.get("attention_factor")
    if attention is None:
        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        attention = mscale(m) / mscale(m_all) if m and m_all else mscale(1.0)
    return inv_freq / factor * ramp + inv_freq * (1 - ramp), float(attention)


def _llama3(inv_freq: torch.Tensor, scaling: dict[str, Any]) -> torch.Tensor:
    """Wavelengths up to a share of the original context stay, those beyond another are stretched by the factor, linear in the
    number of turns between."""
    factor, original, low, high = (float(_needed(scaling, "llama3", key)) for key in (
        "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"))
    turns = original * inv_freq / (2 * math.pi)
    keep = ((turns - low) / (high - low)).clamp(0, 1)
    return inv_freq * (keep + (1 - keep) / factor)


def rotary_inv_freq(
    rotary_dim: int,
    base: float = 10000.0,
    scaling: dict[str, Any] | None = None,
    *,
    seq_len: int | None = None,
    max_position_embeddings: int | None = None,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """``(inv_freq fp64 [rotary_dim / 2], attention_factor)`` for ``tq4_rotary``.

    ``scaling["rope_type"]`` (or ``"type"``): ``default``, ``linear`` (positions divided by ``factor``), ``dynamic`` (the base grows with
    ``seq_len`` beyond ``original_max_position_embeddings``), ``yarn``, ``llama3`` or ``longrope`` (``short_factor`` / ``long_factor`` per
    frequency, by ``seq_len``).  ``max_position_embeddings``: the configuration's longest context, from which ``longrope`` takes the factor
    that its attention factor follows from, where the dictionary holds neither (as those of Phi-3 models do not).

    Raises:
        ValueError: ``rotary_dim`` is not even and positive, the type is unknown, or a key that the type needs is missing (for ``longrope``: all
            that could give its attention factor).
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default")) or "default"
    base = float(scaling.get("rope_theta", base))
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    attention = 1.0
    if kind == "dynamic":
        if rotary_dim == 2:
            raise ValueError("dynamic scaling needs a rotary_dim of 4 or more")
        original = _needed(scaling, kind, "original_max_position_embeddings")
        factor, length = float(_needed(scaling, kind, "factor")), max(seq_len or 0, original)
        base *= (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    inv_freq = base ** -exponent
    if kind == "linear":
        inv_freq = inv_freq / float(_needed(scaling, kind, "factor"))
    elif kind == "yarn":
        inv_freq, attention = _yarn(inv_freq, rotary_dim, base, scaling)
    elif kind == "llama3":
        inv_freq = _llama3(inv_freq, scaling)
    elif kind == "longrope":
        original = _needed(scaling, kind, "original_max_position_embeddings")
        far = seq_len is not None and seq_len > original
        per = torch.tensor(_needed(scaling, kind, "long_factor" if far else "short_factor"), dtype=torch.float64)
        if per.shape != inv_freq.shape:
            raise ValueError(f"longrope needs {inv_freq.numel()} factors, got {per.numel()}")
        inv_freq = inv_freq / per
        attention = scaling.get("attention_factor")
        if attention is None:
            factor = scaling.get("factor")
            if factor is None and max_position_embeddings is None:
                raise ValueError("longrope scaling needs factor, attention_factor or max_position_embeddings")
            factor = float(factor) if factor is not None else max_position_embeddings / original
            attention = 1.0 if factor <= 1 else math.sqrt(1 + math.log(factor) / math.log(original))
    elif kind not in ("default", "dynamic"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    return inv_freq.to(device) if device is not None else inv_freq, float(attention)


__all__ = ["rotary_inv_freq"]
