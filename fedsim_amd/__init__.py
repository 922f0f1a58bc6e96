"""fedsim_amd — MI355X-native server aggregation path for FedSim.

The accelerated path: client vectors are packed into HBM and reduced by a
hand-written gfx950 HIP kernel (libfedagg.so, C-ABI in include/fedagg.h),
bit-identical to the reference CPU aggregation.  Entry points mirror the
reference's names:

  fedsim_amd.utils.SerialAggregator                 (fedsim/utils/aggregators.py)
  fedsim_amd.distributed.centralized.training.FedAvg / AdaBest / FedNova
  fedsim_amd.distributed.centralized.CentralFLAlgorithm

Beside it, operators for training the clients and the server's model on the GPU
(libfedtrain.so, C-ABI in include/fedtrain.h):

  fedsim_amd.functional   linear_act, grouped_linear: differentiable products
                          with fused epilogues, of one model or a cohort
  fedsim_amd.optim        AdamW in one launch, states in 32 or 8 bits
  fedsim_amd.train_ops    the same without autograd
"""
__version__ = "0.1.0"
