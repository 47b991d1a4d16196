from .gram import gram, gram_
from .heads import qk_norm_rope
from .logprobs import PolicyLoss, policy_loss, token_logprobs
from .router import Routing, route

__all__ = ["PolicyLoss", "Routing", "gram", "gram_", "policy_loss", "qk_norm_rope", "route",
           "token_logprobs"]
