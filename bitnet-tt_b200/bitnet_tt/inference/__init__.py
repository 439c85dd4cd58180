"""Generators."""

from .generator_batch32 import Batch32Generator, GenerationStats  # noqa: F401
from .paged_generator import PagedGenerator  # noqa: F401
