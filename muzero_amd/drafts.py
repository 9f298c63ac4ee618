"""Playing ahead of the search: moves drafted by a cheap policy, verified against the search's own.

A cheap policy (a distilled network, or the raw prior) plays several moves ahead; one batched search then evaluates all the
positions it passed through, and `verify_drafts` keeps the drafted moves as far as they are distributed like the search's:
the moves that come out follow the search's policies exactly (mcts/action_selection.py:56-72 is the rule that draws one)."""
from __future__ import annotations

from typing import Optional, Tuple

import numpy as np
import torch

from . import engine as _engine


def verify_drafts(tokens: torch.Tensor, draft: Optional[torch.Tensor], target: torch.Tensor, u_accept: torch.Tensor,
                  u_sample: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keeps drafted move k of a sequence while u_accept[k] * draft[k, x_k] < target[k, x_k]; replaces the first that is not
    kept by a draw from max(target[k] - draft[k], 0) (from target[k] where that is nowhere positive); where all are kept,
    draws one more from the target's next row.

    tokens [B, K] int32 / int64; draft [B, K, V] the probabilities they were drawn from, or None where each was its policy's
    only choice; target [B, K + 1, V] of the same type (float64, float32, bfloat16, float16); u_accept [B, K] and u_sample
    [B] float64 uniforms of [0, 1); lengths int32 [B]: drafted moves of each sequence (None: K).  Sums are float64 and a draw
    takes the first index whose running sum exceeds u * the whole, as np.random.choice does.  Probabilities that are
    negative, infinite or NaN count as 0, a drafted move outside 0..V-1 is not kept.
    Returns (accepted int32 [B], moves [B, K + 1] of the type of tokens: the kept drafts, the drawn move, -1 behind it; a
    target row without any mass yields -1)."""
    where = target.get_device() if torch.is_tensor(target) else -1
    for name, t in (('target', target), ('tokens', tokens), ('draft', draft), ('u_accept', u_accept), ('u_sample', u_sample),
                    ('lengths', lengths)):
        if t is None and name in ('draft', 'lengths'):
            continue
        if not torch.is_tensor(t) or not t.is_cuda:
            raise _engine.EngineError(f'verify_drafts needs device tensors (there is no CPU fallback): {name}')
        if t.get_device() != where:
            raise ValueError(f'verify_drafts: {name} is on another device than the target')
    if tokens.dim() != 2 or target.dim() != 3:
        raise ValueError('verify_drafts: tokens [B, K] and target [B, K + 1, V] expected')
    B, K = tokens.shape
    V = target.shape[2]
    if tuple(target.shape) != (B, K + 1, V) or (draft is not None and tuple(draft.shape) != (B, K, V)) or V < 1:
        raise ValueError(f'verify_drafts: target must be [B, K + 1, V] and draft [B, K, V], got {tuple(target.shape)} and '
                         f'{None if draft is None else tuple(draft.shape)} for {B} x {K} tokens')
    if target.dtype not in _engine.ELEMENT_TYPES or (draft is not None and draft.dtype != target.dtype):
        raise ValueError('verify_drafts: draft and target must share a floating type')
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError('verify_drafts: tokens must be int32 or int64')
    if tuple(u_accept.shape) != (B, K) or tuple(u_sample.shape) != (B,) or u_accept.dtype != torch.float64 or u_sample.dtype != torch.float64:
        raise ValueError('verify_drafts: u_accept [B, K] and u_sample [B] must be float64')
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype != torch.int32):
        raise ValueError('verify_drafts: lengths must be int32 [B]')
    return _engine.torch_calls().verify_drafts(tokens, draft, target, u_accept, u_sample, lengths, _engine.raw_stream(where))


def verify_by_search(mcts, network, observations, legal_actions, to_play, tokens: torch.Tensor, draft: Optional[torch.Tensor],
                     temperature: float = 1.0, lengths: Optional[torch.Tensor] = None, action_encoder=None, seed: int = 0,
                     tree_id0: int = 0) -> Tuple[torch.Tensor, torch.Tensor, np.ndarray]:
    """Moves drafted K ahead in B games against the search's own policies: one `search_batch` over all B * (K + 1) positions
    the drafts passed through, then `verify_drafts` with uniforms drawn from `np.random` behind the search's noise (B * K for
    the drafts, then B for the draws).

    observations [B, K + 1, ...], legal_actions [B, K + 1, A], to_play [B, K + 1]: the position in front of every drafted move
    and the one behind the last (behind a game's own length: any position).  tokens [B, K] device int32 / int64, draft
    [B, K, A] device float64 or None.  `temperature` as for `search_batch`: at 0 a PUCT search's policy is its most visited move
    (shared where several tie), a Gumbel search has none.
    Returns (accepted, moves, root values [B, K + 1])."""
    B, K = tokens.shape
    observations = observations if torch.is_tensor(observations) else np.asarray(observations)
    n = B * (K + 1)
    if tuple(observations.shape[:2]) != (B, K + 1):
        raise ValueError(f'verify_by_search: observations must be [{B}, {K + 1}, ...], got {tuple(observations.shape)}')
    _, values, probs = mcts.search_batch(network, observations.reshape((n,) + tuple(observations.shape[2:])),
                                         np.asarray(legal_actions).reshape(n, -1), np.asarray(to_play).reshape(n), temperature,
                                         action_encoder=action_encoder, seed=seed, tree_id0=tree_id0)
    on = lambda a: torch.as_tensor(np.ascontiguousarray(a, dtype=np.float64), device=tokens.device)  # noqa: E731
    target = on(np.stack([np.asarray(p) for p in probs]) if not isinstance(probs, np.ndarray) else probs).reshape(B, K + 1, -1)
    u_accept, u_sample = np.random.random_sample((B, K)), np.random.random_sample(B)
    accepted, moves = verify_drafts(tokens, draft, target, on(u_accept), on(u_sample), lengths=lengths)
    return accepted, moves, np.asarray(values, dtype=np.float64).reshape(B, K + 1)
