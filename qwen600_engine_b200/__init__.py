"""B200-native token sampler for qwen600_engine.

``sampler`` mirrors the reference's sampler API over the C ABI of
``libqwen600_sampler.so`` (include/qwen600_sampler.h); ``w4`` is the lm_head with
4-bit weights, ``losses`` scores sampled tokens and gives the policy and
preference losses over them with their gradients; ``workloads`` makes the
seeded synthetic logit batches used by the tests and the benchmark.
"""
from . import workloads  # noqa: F401

__version__ = "0.1.0"


def _module(name):
    import importlib
    return importlib.import_module(__name__ + "." + name)


_HOME = {name: "sampler" for name in ("Sampler", "SamplingConfig", "build_sampler", "sample",
                                      "reset_sampler_history", "free_sampler")}
_HOME |= {name: "w4" for name in ("W4Weight", "lm_head_w4")}
_HOME |= {name: "losses" for name in ("token_logprobs", "token_logprobs_backward", "policy_loss",
                                      "preference_loss")}


def __getattr__(name):
    # The CUDA library is loaded on first use so that the synthetic-workload
    # helpers import on machines without the built library.
    if name in ("sampler", "w4", "losses"):
        return _module(name)
    if name in _HOME:
        return getattr(_module(_HOME[name]), name)
    raise AttributeError(name)
