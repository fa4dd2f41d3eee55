"""Callers of the hot path: the DIP / cache-aware DIP MLP drivers, and the paged KV cache of several sequences."""
from . import dip, paged_kv

__all__ = ["dip", "paged_kv"]
