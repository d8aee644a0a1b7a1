"""Python calls of a ragged batch's operators (include/cactus_b200_batch.h).

Thin ctypes plumbing: arrays are addresses in device memory or objects with ``data_ptr()``; strides are
in elements and default to dense rows; None stands for what a call does not have.
"""
from __future__ import annotations

from . import check, lib
from .kv4 import _addr


def add_rms_norm_q8(x, weight, rows: int, dims: int, codes=None, scales=None, normed=None, residual=None, sum=None,
                    eps: float = 1e-6, x_stride: int | None = None, residual_stride: int | None = None,
                    sum_stride: int | None = None, stream: int = 0):
    """Rows x (+ residual, stored in sum), normalised, as int8 codes with a scale each and/or as fp16."""
    check(lib().cactus_cuda_add_rms_norm_q8(_addr(x), x_stride or dims, _addr(residual), residual_stride or dims,
                                            _addr(weight), _addr(sum), sum_stride or dims, _addr(codes), _addr(scales),
                                            _addr(normed), rows, dims, eps, stream), "add_rms_norm_q8")


def lora_plan_bytes(seqs: int, tokens: int, adapters: int) -> int:
    return lib().cactus_cuda_lora_plan_bytes(seqs, tokens, adapters)


def lora_workspace(tokens: int, max_rank: int) -> int:
    return lib().cactus_cuda_lora_workspace(tokens, max_rank)


def lora_plan(token_offsets, adapter_ids, seqs: int, tokens: int, adapters: int, plan, plan_bytes: int, stream: int = 0):
    """Groups a batch's rows by adapter: one plan for all projections of all layers of a step."""
    check(lib().cactus_cuda_lora_plan(_addr(token_offsets), _addr(adapter_ids), seqs, tokens, adapters, _addr(plan),
                                      plan_bytes, stream), "lora_plan")


def lora(x, a, b, output, plan, plan_bytes: int, seqs: int, tokens: int, adapters: int, max_rank: int,
         in_features: int, out_features: int, workspace, workspace_bytes: int, base=None, ranks=None, scales=None,
         x_stride: int | None = None, base_stride: int | None = None, output_stride: int | None = None, stream: int = 0):
    """output = base + scale * (x A^T) B^T, each row with its sequence's adapter."""
    check(lib().cactus_cuda_lora_f16(_addr(x), x_stride or in_features, _addr(a), _addr(b), _addr(ranks), _addr(scales),
                                     _addr(base), base_stride or out_features, _addr(output),
                                     output_stride or out_features, _addr(plan), plan_bytes, seqs, tokens, adapters,
                                     max_rank, in_features, out_features, _addr(workspace), workspace_bytes, stream),
          "lora")


def logits_process(logits, output, rows: int, vocab: int, penalties=None, history=None, history_offsets=None,
                   prompt_lens=None, num_history: int = 0, bias_ids=None, bias_values=None, bias_offsets=None,
                   num_biases: int = 0, masks=None, mask_stride: int | None = None, num_masks: int = 0, mask_ids=None,
                   logits_stride: int | None = None, output_stride: int | None = None, stream: int = 0):
    """Penalties, biases and grammar masks on a batch's logits; output may be logits."""
    check(lib().cactus_cuda_logits_process_f16(
        _addr(logits), logits_stride or vocab, _addr(output), output_stride or vocab, rows, vocab, _addr(penalties),
        _addr(history), _addr(history_offsets), _addr(prompt_lens), num_history, _addr(bias_ids), _addr(bias_values),
        _addr(bias_offsets), num_biases, _addr(masks), mask_stride or (vocab + 31) // 32, num_masks, _addr(mask_ids),
        stream), "logits_process")
