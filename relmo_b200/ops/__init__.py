"""Operator wrappers (mirrors ``relmo.ops``)."""

from . import decoder, mp

__all__ = ["decoder", "mp"]
