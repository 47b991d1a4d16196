"""Kernels as functions on tensors. The row operators are loaded when first asked for: they need
``libmuon_amd_torch.so``, and ``gram`` does not."""

from importlib import import_module

from .gram import gram, gram_

_ROW_OPERATORS = {"PolicyLoss": "logprobs", "Routing": "router", "policy_loss": "logprobs",
                  "qk_norm_rope": "heads", "route": "router", "token_logprobs": "logprobs"}

__all__ = ["PolicyLoss", "Routing", "gram", "gram_", "policy_loss", "qk_norm_rope", "route",
           "token_logprobs"]


def __getattr__(name: str):
    if name not in _ROW_OPERATORS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = getattr(import_module(f"{__name__}.{_ROW_OPERATORS[name]}"), name)
    globals()[name] = value
    return value


def __dir__():
    return sorted({*globals(), *__all__})
