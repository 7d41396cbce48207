"""B200 (sm_100a) fused GRPO / PPO-clip token loss: a drop-in for the loss region of
demon2036/MLLM-JAX's TrainGRPOModule (MLLM_JAX/train_modules/__init__.py:118-180).

Importing the package does not need a GPU or the built library; calling an operator does.
"""
from ._lib import GrpoError, LIB_PATH, launch_count  # noqa: F401
from .ops import (  # noqa: F401
    LossConfig,
    TokenLossProblem,
    grpo_token_loss,
    grpo_token_loss_flat,
    grpo_value_and_grad,
    sft_cross_entropy,
    token_logprobs,
)
from .embedding import embedding_grad, embedding_lookup  # noqa: F401
from .fp8 import Fp8Blocks, fp8_matmul, quantize_fp8  # noqa: F401
from .linear_loss import linear_grpo_value_and_grad, lm_head_forward  # noqa: F401
from .preference import (  # noqa: F401
    PreferenceConfig,
    preference_logps_value_and_grad,
    preference_loss,
    preference_loss_from_logps,
    preference_value_and_grad,
)
from .train_module import (  # noqa: F401
    TrainGRPOModule,
    per_sample_entropy,
    ppo_actor_critic_terms,
    ppo_policy_terms,
    ppo_value_loss,
)

__all__ = [
    "Fp8Blocks", "GrpoError", "LIB_PATH", "LossConfig", "PreferenceConfig", "TokenLossProblem", "TrainGRPOModule",
    "embedding_grad", "embedding_lookup", "fp8_matmul", "grpo_token_loss", "grpo_token_loss_flat",
    "grpo_value_and_grad", "launch_count", "linear_grpo_value_and_grad", "lm_head_forward", "per_sample_entropy",
    "ppo_actor_critic_terms", "ppo_policy_terms", "ppo_value_loss", "preference_logps_value_and_grad",
    "preference_loss", "preference_loss_from_logps", "preference_value_and_grad", "quantize_fp8",
    "sft_cross_entropy",
    "token_logprobs",
]
