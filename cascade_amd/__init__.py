"""cascade_amd: MI355X (gfx950) per-partition suffix sort by prefix doubling, behind a C ABI, and operators of a language model
over the same token texts.

The compute lives in libcascade_hip.so (hand-written HIP, include/cascade_hip.h) and libcascade_lm.so (include/cascade_lm.h); this
package is the thin host-side mirror of the reference's builder interface for the sort, and the operators on torch tensors.
"""
from . import _native, workloads
from .gpu_saca import GPU_SACA, PartitionSorter, output_cut, pack_keys, partition_ids, sort_partition, sort_partitions, stage_slab
from .language_model import (add_norm, attend, clip_gradients, distillation_loss, embed, embed_tokens, embed_tokens_backward, linear_cross_entropy,
                             linear_cross_entropy_backward, linear_distillation, linear_distillation_backward, next_token_loss, residual_norm, residual_norm_backward,
                             span_attention, span_attention_backward, token_spans)

__all__ = ["GPU_SACA", "PartitionSorter", "output_cut", "pack_keys", "partition_ids", "sort_partition", "sort_partitions", "stage_slab", "workloads", "_native",
           "add_norm", "attend", "clip_gradients", "distillation_loss", "embed", "embed_tokens", "embed_tokens_backward", "linear_cross_entropy",
           "linear_cross_entropy_backward", "linear_distillation", "linear_distillation_backward", "next_token_loss", "residual_norm", "residual_norm_backward", "span_attention", "span_attention_backward", "token_spans"]
