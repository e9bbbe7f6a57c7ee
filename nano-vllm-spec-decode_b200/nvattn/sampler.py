"""Token sampling and speculative verify (nanovllm/layers/sampler.py).

verify_drafts_greedy(logits, draft_token_ids, num_drafts) returns what verify_drafts returns when every
temperature is 0: the target ids are the row argmaxes of logits [S*(K+1), V] (torch's argmax, first index of the
maximum, as sampler.py:66), and the accept length and next token come from the integer kernel behind
ops.greedy_accept (sampler.py:67, 79-82).  Unlike the reference it reads no device value on the host (the
reference's all-greedy test at sampler.py:64 syncs), so a verify step stays capturable in a CUDA graph.

The random branches take their random numbers as arguments (uniform numbers, one per drawn token and one per draft),
so that a step is a function of its inputs and stays capturable in a CUDA graph:

  sample_tokens(logits, temperatures, uniforms, top_k, top_p, min_p)      Sampler.forward (sampler.py:7-16), with
                                                                          top-k, top-p and min-p
  verify_drafts_sampled(logits, draft_token_ids, num_drafts, temperatures, accept_uniforms, uniforms, ...)
                                                                          verify_drafts (sampler.py:28-103) with
                                                                          temperatures, for drafts that are fixed
                                                                          tokens (n-gram, greedy draft model)

Rows with a temperature of 0 are greedy in both.
"""
import torch

from . import ops
from .ops import sample_tokens  # noqa: F401


def verify_drafts_greedy(logits: torch.Tensor, draft_token_ids: torch.Tensor, num_drafts: torch.Tensor):
    """logits [S*(K+1), V], draft_token_ids [S, K], num_drafts [S] -> (num_accepted [S], next_token [S]) int64,
    the dtype the reference returns.  Sequence s keeps draft_token_ids[s, :num_accepted[s]], then next_token[s]."""
    S, K = draft_token_ids.shape
    top1 = logits.view(S, K + 1, logits.size(-1)).argmax(dim=-1)    # [S, K+1] int64
    return ops.greedy_accept(top1, draft_token_ids.to(top1.dtype), num_drafts.to(top1.dtype))


def verify_drafts_sampled(logits: torch.Tensor, draft_token_ids: torch.Tensor, num_drafts: torch.Tensor,
                          temperatures: torch.Tensor, accept_uniforms: torch.Tensor, uniforms: torch.Tensor,
                          top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                          min_p: torch.Tensor | None = None):
    """verify_drafts with temperatures: logits [S*(K+1), V] (bf16 or float32), draft_token_ids [S, K] and num_drafts [S]
    (integers), temperatures / uniforms / settings [S], accept_uniforms [S, K] -> (num_accepted [S], next_token [S])
    int64.  Sequence s keeps draft_token_ids[s, :num_accepted[s]], then next_token[s]; what comes out is distributed as
    if every token had been drawn by sample_tokens."""
    if draft_token_ids.dtype is not torch.int64 or num_drafts.dtype is not torch.int64:
        draft_token_ids, num_drafts = draft_token_ids.to(torch.int64), num_drafts.to(torch.int64)
    return ops.verify_sampled(logits, draft_token_ids, num_drafts, temperatures, accept_uniforms, uniforms, top_k, top_p,
                              min_p)
