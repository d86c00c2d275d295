"""Alias of feather_amd.routines.paged_cache."""
from feather_amd.routines.paged_cache import *  # noqa: F401,F403
