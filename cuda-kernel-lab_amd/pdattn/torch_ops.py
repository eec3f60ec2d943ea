"""PyTorch operators over the C ABI, for use from a serving stack.

``torch.ops.pdattn.paged_decode`` runs the balanced decode path (pdattn_plan_run) and
``torch.ops.pdattn.append_kv`` the paged KV append (pdattn_append_kv). ``rope_append_kv``,
``tree_attention`` and ``accept_kv`` are the step of a decoder that checks drafted tokens
(pdattn_rope_append_kv, pdattn_tree_attention, pdattn_accept_kv): rotate and append the drafted rows,
attend from them, move the accepted ones to the front. All launch on the current stream of their
tensors' device. They are registered with ``torch.library.custom_op``, with fake (shape-only)
implementations, so they trace under torch.compile and work with torch's stream and graph
machinery. The arithmetic is the library's: these functions only pass tensors through.

The balanced plan is built on the host from host copies of kv_indptr and kv_last_page_len
(``indptr_host`` / ``last_host``, int32 CPU tensors), the way FlashInfer's plan() works. Plans and
their workspaces are cached by the contents of those tables, so a decode loop over one batch
composition plans once.
"""
from __future__ import annotations

from collections import OrderedDict

import torch

from . import (HEAD_DIM, Plan, Workspace, accept_kv as _accept_kv, append_kv as _append_kv, make_rope_append_params,
               make_tree_params, rope_append_kv as _rope_append_kv, tree_attention as _tree_attention, tree_workspace_size)

_PLAN_CACHE_SIZE = 8
_plans: "OrderedDict[tuple, tuple]" = OrderedDict()


def _plan_for(indptr_host: torch.Tensor, last_host: torch.Tensor, Hq: int, Hkv: int,
              device: torch.device):
    ip = indptr_host.to(torch.int32).contiguous()
    la = last_host.to(torch.int32).contiguous()
    key = (ip.numpy().tobytes(), la.numpy().tobytes(), Hq, Hkv, device.index)
    hit = _plans.get(key)
    if hit is not None:
        _plans.move_to_end(key)
        return hit
    B = ip.numel() - 1
    plan = Plan(ip.numpy(), la.numpy(), B, Hq, Hkv)
    ws = torch.empty(max(256, plan.workspace_bytes), dtype=torch.uint8, device=device)
    plan.upload(ws, ws.numel(), torch.cuda.current_stream(device))
    _plans[key] = (plan, ws)
    if len(_plans) > _PLAN_CACHE_SIZE:
        _, (old_plan, _) = _plans.popitem(last=False)
        old_plan.close()
    return plan, ws


@torch.library.custom_op("pdattn::paged_decode", mutates_args=())
def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                 indptr_host: torch.Tensor, last_host: torch.Tensor,
                 sm_scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Paged GQA decode attention. q [B, Hq, 128] fp16; k_cache / v_cache [num_pages, 16, Hkv,
    128] fp16; kv_indptr [B+1], kv_indices [nnz], kv_last_page_len [B] int32 on the device, and
    host copies of kv_indptr / kv_last_page_len. Returns (out [B, Hq, 128] fp16, lse [B, Hq] fp32,
    the natural log of the scaled scores)."""
    if q.dtype != torch.float16 or k_cache.dtype != torch.float16 or v_cache.dtype != torch.float16:
        raise TypeError("q, k_cache and v_cache must be float16")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or k_cache.dim() != 4 or k_cache.shape[3] != HEAD_DIM:
        raise ValueError("q must be [B, Hq, 128] and the caches [num_pages, 16, Hkv, 128]")
    B, Hq = q.shape[0], q.shape[1]
    Hkv = k_cache.shape[2]
    if indptr_host.numel() != B + 1 or last_host.numel() != B:
        raise ValueError("host page-table copies do not match the batch size")
    q = q.contiguous()
    plan, ws = _plan_for(indptr_host, last_host, Hq, Hkv, q.device)
    out = torch.empty_like(q)
    lse = torch.empty(B, Hq, dtype=torch.float32, device=q.device)
    plan.run(q, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, out, lse, ws, ws.numel(),
             sm_scale=sm_scale, stream=torch.cuda.current_stream(q.device))
    return out, lse


@paged_decode.register_fake
def _paged_decode_fake(q, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, indptr_host,
                       last_host, sm_scale):
    return torch.empty_like(q), q.new_empty((q.shape[0], q.shape[1]), dtype=torch.float32)


@torch.library.custom_op("pdattn::append_kv", mutates_args=("k_cache", "v_cache"))
def append_kv(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
              batch_idx: torch.Tensor, positions: torch.Tensor) -> None:
    """Write k_new / v_new [n, Hkv, 128] fp16 into the paged caches at (batch_idx[t],
    positions[t]); the page table already covers the appended tokens."""
    if k_new.dtype != torch.float16 or k_cache.dtype != torch.float16:
        raise TypeError("K/V rows and caches must be float16")
    B = kv_indptr.numel() - 1
    _append_kv(k_new.contiguous(), v_new.contiguous(), k_cache, v_cache, kv_indptr, kv_indices,
               batch_idx, positions, B, k_cache.shape[2],
               stream=torch.cuda.current_stream(k_cache.device))


@append_kv.register_fake
def _append_kv_fake(k_new, v_new, k_cache, v_cache, kv_indptr, kv_indices, batch_idx, positions):
    return None


def _check_tables(device, **tables):
    """int32, contiguous and on the device; those with a length, of it."""
    for name, (x, n) in tables.items():
        if x is None:
            continue
        if x.dtype != torch.int32 or x.device != device or not x.is_contiguous():
            raise TypeError(f"{name} must be contiguous int32 on {device}")
        if n is not None and x.numel() != n:
            raise ValueError(f"{name} has {x.numel()} elements, not {n}")


def _check_caches(k_cache, v_cache):
    for x in (k_cache, v_cache):
        if x.dtype != torch.float16:
            raise TypeError("the caches must be float16")
        if x.dim() != 4 or x.shape[1] != 16 or x.shape[3] != HEAD_DIM or not x.is_contiguous():
            raise ValueError("the caches must be contiguous [num_pages, 16, Hkv, 128]")
    if k_cache.shape != v_cache.shape or k_cache.device != v_cache.device:
        raise ValueError("the caches must be alike")


@torch.library.custom_op("pdattn::rope_append_kv", mutates_args=("k_cache", "v_cache"))
def rope_append_kv(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   kv_indptr: torch.Tensor, kv_indices: torch.Tensor, batch_idx: torch.Tensor, positions: torch.Tensor,
                   freq: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
                   rope_positions: torch.Tensor | None = None) -> torch.Tensor:
    """Rotated q [n, Hq, 128]; k_new, rotated, and v_new [n, Hkv, 128] are written into the paged caches at (batch_idx[t],
    positions[t]). freq: float64 [rotary_dim / 2] (pdattn.rope_frequencies). The angles are those of rope_positions where they
    are given. q, k_new and v_new may be slices of one projection's output."""
    _check_caches(k_cache, v_cache)
    if any(x.dtype != torch.float16 or x.device != k_cache.device for x in (q, k_new, v_new)) or freq.dtype != torch.float64:
        raise TypeError("q, k_new and v_new must be float16 on the caches' device, freq float64")
    if freq.device != k_cache.device or not freq.is_contiguous() or k_new.dim() != 3 or k_new.shape[1] != k_cache.shape[2]:
        raise ValueError("freq must be contiguous on the caches' device, k_new [n, Hkv, 128]")
    n, B = k_new.shape[0], kv_indptr.numel() - 1
    _check_tables(k_cache.device, kv_indptr=(kv_indptr, None), kv_indices=(kv_indices, None), batch_idx=(batch_idx, n),
                  positions=(positions, n), rope_positions=(rope_positions, n))
    q_out = q.new_empty(q.shape)
    p = make_rope_append_params(q, k_new, v_new, q_out, k_cache, v_cache, kv_indptr, kv_indices, batch_idx, positions, freq, B,
                                rotary_dim=2 * freq.numel(), interleaved=interleaved, scale=scale, rope_positions=rope_positions)
    with torch.cuda.device(k_cache.device):
        _rope_append_kv(p, torch.cuda.current_stream(k_cache.device))
    return q_out


@rope_append_kv.register_fake
def _rope_append_kv_fake(q, k_new, v_new, k_cache, v_cache, kv_indptr, kv_indices, batch_idx, positions, freq, interleaved=False,
                         scale=1.0, rope_positions=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("pdattn::tree_attention", mutates_args=())
def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_indptr: torch.Tensor,
                   kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, sm_scale: float,
                   q_indptr: torch.Tensor | None = None, max_tokens: int = 1, mask: torch.Tensor | None = None,
                   depth: torch.Tensor | None = None, soft_cap: float = 0.0, slopes: torch.Tensor | None = None,
                   window: int = 0, sink: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of each sequence's newest tokens, already in the cache, over the paged cache. q [n_tokens, Hq, 128] fp16;
    q_indptr [B + 1]: their rows of q (none: one token a sequence); mask int32 [n_tokens, words], the drafted tokens that each
    sees, as bits (none: chains); depth: the tokens' positions behind the context. Scores may be capped, biased by
    distance (slopes, fp32 [Hq]) and cut to a window with the first `sink` keys kept. Returns (out [n_tokens, Hq, 128] fp16,
    lse [n_tokens, Hq] fp32); rows behind the last sequence's are 0 and minus infinity."""
    _check_caches(k_cache, v_cache)
    if q.dtype != torch.float16 or q.device != k_cache.device:
        raise TypeError("q must be float16 on the caches' device")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError("q must be [n_tokens, Hq, 128]")
    n, Hq, B, Hkv = q.shape[0], q.shape[1], kv_last_page_len.numel(), k_cache.shape[2]
    if q_indptr is None and n != B:
        raise ValueError("without q_indptr q has one row per sequence")
    if mask is not None and (mask.dim() != 2 or mask.shape[0] != n):
        raise ValueError("mask must be [n_tokens, words]")
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.numel() != Hq or slopes.device != q.device or not slopes.is_contiguous()):
        raise ValueError("slopes must be contiguous float32 [Hq]")
    _check_tables(q.device, kv_indptr=(kv_indptr, B + 1), kv_indices=(kv_indices, None), kv_last_page_len=(kv_last_page_len, B),
                  q_indptr=(q_indptr, B + 1), mask=(mask, None), depth=(depth, n))
    if kv_indices.numel() == 0 or k_cache.numel() == 0:   # no key anywhere
        return torch.zeros_like(q, memory_format=torch.contiguous_format), q.new_full((n, Hq), float("-inf"), dtype=torch.float32)
    q = q.contiguous()
    p = make_tree_params(q, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, B, Hq, Hkv, q_indptr=q_indptr,
                         max_tokens=max_tokens, mask=mask, depth=depth, sm_scale=sm_scale, soft_cap=soft_cap, slopes=slopes,
                         window=window, sink=sink)
    out = torch.zeros_like(q) if q_indptr is not None else torch.empty_like(q)
    lse = q.new_full((n, Hq), float("-inf"), dtype=torch.float32) if q_indptr is not None else q.new_empty((n, Hq), dtype=torch.float32)
    with torch.cuda.device(q.device):
        space = torch.empty(max(256, tree_workspace_size(p)), dtype=torch.uint8, device=q.device)
        _tree_attention(p, out, lse, Workspace(space.data_ptr(), space.numel(), 0), torch.cuda.current_stream(q.device))
    return out, lse


@tree_attention.register_fake
def _tree_attention_fake(q, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, sm_scale, q_indptr=None, max_tokens=1,
                         mask=None, depth=None, soft_cap=0.0, slopes=None, window=0, sink=0):
    return q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[1]), dtype=torch.float32)


@torch.library.custom_op("pdattn::accept_kv", mutates_args=("k_cache", "v_cache"))
def accept_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
              kv_last_page_len: torch.Tensor, q_indptr: torch.Tensor, accepted_indptr: torch.Tensor,
              accepted: torch.Tensor) -> None:
    """The rows of each sequence's accepted drafted tokens (ascending, accepted[accepted_indptr[b] ..]) moved to the front of
    its drafted range in the caches."""
    _check_caches(k_cache, v_cache)
    B = kv_last_page_len.numel()
    _check_tables(k_cache.device, kv_indptr=(kv_indptr, B + 1), kv_indices=(kv_indices, None),
                  kv_last_page_len=(kv_last_page_len, B), q_indptr=(q_indptr, B + 1), accepted_indptr=(accepted_indptr, B + 1),
                  accepted=(accepted, None))
    if accepted.numel() == 0 or kv_indices.numel() == 0:   # nothing to move
        return
    with torch.cuda.device(k_cache.device):
        _accept_kv(k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, q_indptr, accepted_indptr, accepted, B,
                   k_cache.shape[2], stream=torch.cuda.current_stream(k_cache.device))


@accept_kv.register_fake
def _accept_kv_fake(k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, q_indptr, accepted_indptr, accepted):
    return None
