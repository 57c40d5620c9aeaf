"""B200-native Kimi Delta Attention: hand-written sm_100a kernels behind a C ABI
(include/kda_b200.h) and a host-side mirror of the reference mixer interface."""

from .attention import PagedAttention, PagedCache, paged_attention, qk_norm_rope, qk_norm_rope_append
from .kda import (KDAState, KimiDeltaAttention, RMSNormGated, ShortConvolution, chunk_kda, chunk_kda_norm, k3_decay_gate, kda,
                  kda_backend_provenance, prepare_kda_backend, recurrent_kda_step, short_convolutions)

__all__ = ["KDAState", "KimiDeltaAttention", "PagedAttention", "PagedCache", "RMSNormGated", "ShortConvolution", "chunk_kda", "chunk_kda_norm", "k3_decay_gate", "kda",
           "kda_backend_provenance", "paged_attention", "prepare_kda_backend", "qk_norm_rope", "qk_norm_rope_append", "recurrent_kda_step", "short_convolutions"]
