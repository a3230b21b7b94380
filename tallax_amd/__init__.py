"""tallax_amd: MI355X-native (gfx950 HIP) sort / select / sample path of tallax.

Public modules mirror the reference: `tax` (tallax/tax.py), `tumpy`
(tallax/tumpy.py) and `sampling` (tallax/_src/sampling.py); `kvcache`,
`speculative` and `experts` are the parts of a serving step around the sampler
that the reference leaves to its caller.
"""
from . import experts, kvcache, prefill, sampling, speculative, tax, tumpy  # noqa: F401

__all__ = ["tax", "tumpy", "sampling", "prefill", "kvcache", "speculative", "experts"]
