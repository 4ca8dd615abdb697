from .dp_rnn import DPGRU, DPLSTM, DPRNNBase, RNNLinear
from .dp_multihead_attention import DPMultiheadAttention, SequenceBias
from .dp_rms_norm import DPRMSNorm, rms_norm
from .dp_selective_ssm import (DPCausalConv, DPSelectiveScan, DPSelectiveSSM, DPSelectiveSSMBlock, SSMLinear, SSMState, causal_conv,
                            causal_conv_step, selective_scan, selective_scan_step)

__all__ = ["DPGRU", "DPLSTM", "DPRNNBase", "RNNLinear", "DPMultiheadAttention", "SequenceBias", "DPRMSNorm", "rms_norm",
           "DPCausalConv", "DPSelectiveScan", "DPSelectiveSSM", "DPSelectiveSSMBlock", "SSMLinear", "SSMState", "causal_conv",
           "causal_conv_step", "selective_scan", "selective_scan_step"]
from .fused_gru import FusedLinearCellGRU, fuse_recurrences, run_together
