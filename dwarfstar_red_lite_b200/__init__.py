"""redcuda: B200 (sm_100a) backend for the Qwen3-Next decode hot path of Red Lite.

The compute lives in libredcuda.so (hand-written CUDA behind the C ABI of include/redcuda.h); this package is the
thin Python host mirror of that ABI plus seeded synthetic inputs. There is no CPU path: every operation raises when
the library or a CUDA device is missing.
"""
from . import synth  # noqa: F401
from .redcuda import (DeltaDims, MoeLayer, PagedKv, RedcudaError, delta_rule, delta_rule_device, delta_step_device, deltanet_step, device_status, lib,  # noqa: F401
                      nib_dequant_rows, quant_dequant_rows, quant_matmul_tc, quant_matvec, router_select_softmax_topk, set_codebooks, token_logprobs, token_logprobs_device)
