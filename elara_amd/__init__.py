"""elara_amd: MI355X-native (gfx950) sparse-update path of ELARA.

Hand-written HIP kernels behind a C-ABI (include/elara_amd.h, libelara_amd.so), exposed with the reference's op
signatures:
  elara_amd.ops        gpu_adam, ext().adam_scalars                       (srm2/ops.py)
  elara_amd.gpu_ops    init_rows, replay_rows, ScalarTable                 (srm2/gpu_ops.py)
  elara_amd.logprobs   token_logprobs and its gradient                     (no counterpart)
  elara_amd.norms      rms_norm, rms_norm_fp8 and the backward, from an int8 stream too   (no counterpart)
  elara_amd.gradnorm   grad_norm, clip_grad_norm                           (no counterpart)
  elara_amd.int8       rows in 8-bit integers: quantize, dequantize, linear, weight_grad  (no counterpart)
  elara_amd.sampling   sample_tokens                                       (no counterpart)
"""
__version__ = '0.1.0'
