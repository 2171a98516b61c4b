"""Value estimators on the MI355X kernels: the modules of torchrl.objectives.value (same names), the functional
entry points (``functional``), the cross-GPU statistics exchange, and what a policy over tokens needs beside them: processed logits,
log-probabilities of the stored tokens, activations kept in 8 bits."""
from torchrl_amd.objectives.value import functional  # noqa: F401
from torchrl_amd.objectives.value.advantages import GAE, TDLambdaEstimate, TDLambdaEstimator, VTrace  # noqa: F401
from torchrl_amd.objectives.value.advantages import TD0Estimate, TD0Estimator, TD1Estimate, TD1Estimator  # noqa: F401
from torchrl_amd.objectives.value.advantages import KeyedModule, RolloutData, ValueEstimatorBase  # noqa: F401
from torchrl_amd.objectives.value.stats_exchange import StatsExchange  # noqa: F401,E402
from torchrl_amd.objectives.value.kept_activations import (CheckpointedLinear, QuantizedActivation, checkpointed_linear,  # noqa: F401
                                                           quantize_activation)
from torchrl_amd.objectives.value.tokens import TokenActor, process_logits, token_log_prob  # noqa: F401

__all__ = ["functional", "GAE", "TDLambdaEstimator", "TDLambdaEstimate", "VTrace", "TD0Estimator", "TD0Estimate",
           "TD1Estimator", "TD1Estimate", "ValueEstimatorBase", "KeyedModule", "RolloutData", "StatsExchange",
           "process_logits", "token_log_prob", "TokenActor", "quantize_activation", "QuantizedActivation", "checkpointed_linear",
           "CheckpointedLinear"]
