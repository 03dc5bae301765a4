"""oal_amd: MI355X (gfx950) HIP implementation of OAL grouped quadratic attention.

Drop-in for the reference ``oal_attention`` operator surface:

* ``oal_amd.oal_attention`` (``oal_attention.oal_attention``)
* ``oal_amd.hd_attention.grouped_causal_attention``
* ``oal_amd.hd_block_gemm_adapters.prepare_grouped_hd_block_gemm`` /
  ``run_prepared_grouped_hd_block_gemm``
* ``oal_amd.hd_block_gemm_autograd._HDParallelBlockGemmFunction``
* ``oal_amd.hd_block_gemm.build_hd_block_gemm_plan`` / ``canonical_pair_layout``

Beside it, for whole sequences and token by token:

* ``oal_amd.gated_delta.gated_delta_attention`` / ``gated_delta_step``
* ``oal_amd.decay_attention.decay_attention`` / ``decay_step``
* ``oal_amd.window_attention.window_attention`` / ``window_attention_step`` / ``window_cache``

Around them:

* ``oal_amd.norm_rotary.norm_rotary_heads``
* ``oal_amd.token_scores.token_log_probs``

The arithmetic runs in ``liboal_amd.so`` (hand-written HIP kernels behind the
C ABI in ``include/oal_amd.h``); PyTorch supplies device memory and streams.
"""

from .grouped_quadratic import oal_attention

__all__ = ["oal_attention"]
