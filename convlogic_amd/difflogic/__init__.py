from .activation_codes import ActivationCodes, decode_activations, encode_activations
from .compiled_model import CompiledLogicNet
from .difflogic import GroupSum, LogicLayer, LogicLayerCudaFunction
from .functional import GradFactor, bin_op, bin_op_s, get_unique_connections
from .losses import balance_loss, distillation_loss, gate_balance, group_cross_entropy, top_logits
from .packbitstensor import PackBitsTensor

__all__ = ["LogicLayer", "GroupSum", "LogicLayerCudaFunction", "PackBitsTensor", "GradFactor", "bin_op", "bin_op_s",
           "get_unique_connections", "CompiledLogicNet", "top_logits", "distillation_loss", "balance_loss", "gate_balance", "group_cross_entropy", "ActivationCodes", "encode_activations",
           "decode_activations"]
