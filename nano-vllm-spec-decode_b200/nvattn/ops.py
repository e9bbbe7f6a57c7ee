"""Torch-facing wrappers over the C ABI, with the signatures of the calls nano-vllm makes on its attention path.

  store_kvcache(key, value, k_cache, v_cache, slot_mapping)        nanovllm/layers/attention.py:33-40
  flash_attn_with_kvcache(q, k_cache, v_cache, cache_seqlens=, block_table=, softmax_scale=, causal=True)
                                                                    flash-attn call at attention.py:75-77
  flash_attn_varlen_func(q, k, v, max_seqlen_q=, cu_seqlens_q=, max_seqlen_k=, cu_seqlens_k=, softmax_scale=,
                         causal=True, block_table=)                 flash-attn call at attention.py:67-70
  greedy_accept(target_ids, draft_ids, num_drafts)                  greedy core of verify_drafts, sampler.py:66-82

The first three also take an 8-bit cache: float8_e4m3fn k_cache / v_cache with k_scale= / v_scale= (float32
[NB, KVH, BS / G], a power of two for each block of G consecutive slots and kv head; kvcache_scales() makes them).

Every op runs on the caller's current CUDA stream, allocates only its output and never syncs (but for the first call of
a size, which allocates).  The attention ops keep one workspace per device and stream and one per device for captured
graphs (split-KV partials and the merge tickets, see _workspace); there is no CPU path: non-CUDA tensors raise.
"""
import contextlib
import threading

import torch

from . import _lib


def _stream() -> int:
    """The current device's current stream (its number alone: a Stream object costs 3 us more a call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The context in which `device` is the current one (nothing to do when it already is)."""
    index = device.index
    if index is None or index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("nvattn ops run on CUDA tensors only (no CPU fallback)")


# The attention workspaces in use, per device index i:
#   i             of calls on the default stream
#   (i, stream)   of calls on another stream (its number)
#   (i, _GRAPH)   of captured calls
# Earlier (smaller) ones stay referenced because captured CUDA graphs hold their addresses.
_WORKSPACES: dict = {}
_RETIRED: list[torch.Tensor] = []
_GRAPH = "graph"
_OWN = threading.local()    # .workspace: the one that this thread's calls are to use (own_workspace)

# Held from taking a workspace to the end of the call that uses it: a call is up to four kernels that pass pieces and a
# plan on through its workspace, and another host thread's on the same stream must not come between them (ctypes lets
# other threads run during a call).
_CALL = threading.RLock()


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _grow(key, nbytes: int, device: torch.device) -> torch.Tensor:
    """The workspace under `key`, allocated zero-filled if there is none of that size."""
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _RETIRED.append(ws)
        ws = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device=device)
        if isinstance(key, tuple) and key[1] is _GRAPH and ws.is_cuda:
            torch.cuda.current_stream(device).synchronize()   # a replay may run on any stream: filled before it can
        _WORKSPACES[key] = ws
    return ws


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """The decode / varlen workspace of a call.  Its merge-ticket words must be zero when a call starts and every
    call leaves them zero, so it is allocated zero-filled once (grown, zero-filled, when a call needs more) and then
    reused.  Calls that may overlap must not share one: each stream has its own, and captured calls use another one of
    the device, whatever stream their graph is replayed on.  Graphs share that one and are replayed one after another
    (as those that share a memory pool are); a graph that is replayed beside others is captured inside own_workspace.
    (Not a workspace per capturing stream: torch hands the same 32 streams out again and again.)  Growing a
    workspace while a CUDA graph is being captured would allocate from the graph's pool and record the zero-fill into
    every replay, so that raises instead: size it first with reserve_workspace (the nano-vllm drop-in does so when the
    KV cache is allocated) or an eager call."""
    own = getattr(_OWN, "workspace", None)
    if own is not None:
        if own.numel() < nbytes or own.device != device:
            raise RuntimeError(f"nvattn: a call on {device} that needs {nbytes} bytes inside own_workspace of "
                               f"{own.numel()} bytes on {own.device}")
        return own
    idx = device.index if device.index is not None else torch.cuda.current_device()
    stream = _raw_stream(idx)
    if stream != 0 and torch.cuda.is_current_stream_capturing():
        ws = _WORKSPACES.get((idx, _GRAPH))
        if ws is None or ws.numel() < nbytes:
            raise RuntimeError(f"nvattn: the attention workspace of cuda:{idx} must grow to {nbytes} bytes during a "
                               "CUDA graph capture; call nvattn.ops.reserve_workspace(...) before capturing")
        return ws
    key = (idx, stream) if stream != 0 else idx
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = _grow(key, nbytes, device)
        _grow((idx, _GRAPH), nbytes, device)
    return ws


def workspace_bytes(max_num_seqs: int, max_num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int = 128,
                    fp8_cache: bool = False) -> int:
    """Bytes of workspace that every decode / verify / varlen call of up to max_num_seqs sequences and max_num_tokens
    query rows fits in on the current device; with fp8_cache, also calls over an 8-bit cache."""
    lib = _lib.load()
    need = max(lib.nva_varlen_workspace_bytes(max_num_seqs, max_num_tokens, num_heads, num_kv_heads, head_dim),
               max(lib.nva_paged_decode_workspace_bytes(max_num_seqs, n, num_heads, num_kv_heads, head_dim)
                   for n in range(1, 49)))
    if fp8_cache:
        need = max(need, lib.nva_paged_attention_fp8_workspace_bytes(max_num_tokens, num_heads, num_kv_heads, head_dim))
    return need


def reserve_workspace(max_num_seqs: int, max_num_tokens: int, num_heads: int, num_kv_heads: int,
                      head_dim: int = 128, device: torch.device | None = None, fp8_cache: bool = False) -> int:
    """Allocate (zero-filled) the workspace every later decode / verify / varlen call of up to max_num_seqs
    sequences and max_num_tokens query rows needs on `device`, so that no call on the current stream, and no captured
    one, allocates; with fp8_cache, also for calls over an 8-bit cache.  Returns its size in bytes.  nano-vllm:
    max_num_seqs and max_num_batched_tokens of its Config."""
    device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    with _on(device), _CALL:
        need = workspace_bytes(max_num_seqs, max_num_tokens, num_heads, num_kv_heads, head_dim, fp8_cache)
        return _workspace(need, device).numel()


@contextlib.contextmanager
def own_workspace(workspace: torch.Tensor):
    """Attention calls that this thread makes inside use `workspace`: uint8, zero-filled once, of workspace_bytes(...).
    For a CUDA graph that is replayed beside other graphs: capture it inside, with a workspace of its own that lives as
    long as the graph does and is filled before the first replay."""
    _need_cuda(workspace)
    assert workspace.dtype == torch.uint8 and workspace.is_contiguous()
    before = getattr(_OWN, "workspace", None)
    _OWN.workspace = workspace
    try:
        yield
    finally:
        _OWN.workspace = before


def reset_workspaces() -> None:
    """Zero-fill every workspace again.  A call that gave up on a pipeline wait (bit 2 of the device error word) may
    leave merge tickets non-zero, after which later calls could merge split pieces wrongly; call this (outside any
    graph capture, with no call in flight, after clearing the error word) before going on.  Those given to own_workspace
    are the caller's to fill."""
    for ws in list(_WORKSPACES.values()) + _RETIRED:
        ws.zero_()


SCALE_BLOCKS = (8, 16, 32, 64, 128, 256)   # tokens per scale of an 8-bit cache (include/nvattn.h)


def kvcache_scales(k_cache: torch.Tensor, scale_block: int = 16):
    """Zero-filled (k_scale, v_scale) for an 8-bit cache [NB, BS, KVH, 128]: one scale for each block of scale_block
    consecutive slots and kv head, set by store_kvcache.  16 costs 0.2% of the cache's bytes; a larger block has less
    to read and rounds again more rows when a louder token joins it."""
    NB, BS, KVH, _ = k_cache.shape
    assert scale_block in SCALE_BLOCKS and BS % scale_block == 0
    return tuple(torch.zeros(NB, KVH, BS // scale_block, dtype=torch.float32, device=k_cache.device) for _ in range(2))


def _scale_block(k_cache, v_cache, k_scale, v_scale) -> int:
    """Checks an 8-bit cache against its scales; returns the tokens per scale."""
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn, "k_scale / v_scale go with a float8_e4m3fn cache"
    assert k_scale is not None and v_scale is not None, "an 8-bit cache needs both k_scale and v_scale"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape
    NB, BS, KVH, _ = k_cache.shape
    assert k_scale.dtype == v_scale.dtype == torch.float32
    assert k_scale.is_contiguous() and v_scale.is_contiguous() and k_scale.shape == v_scale.shape
    blocks = k_scale.shape[-1]
    assert k_scale.shape == (NB, KVH, blocks) and blocks > 0 and BS % blocks == 0, "scales are [NB, KVH, BS / G]"
    assert BS // blocks in SCALE_BLOCKS
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert k_cache.device == v_cache.device == k_scale.device == v_scale.device
    return BS // blocks


def _row_stride(x: torch.Tensor) -> int:
    """The row stride of a matrix, for the C ABI, which refuses rows that overlap (an expanded view's are 0 apart).  A
    single row has no stride to speak of: its width, whatever the view says."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _is_fp8(k_cache, k_scale, v_scale) -> bool:
    return k_scale is not None or v_scale is not None or k_cache.dtype == torch.float8_e4m3fn


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None) -> None:
    """Scatter this step's K/V rows into the paged cache (attention.py:33-40; same asserts).

    With a float8_e4m3fn cache and its scales the bf16 rows are rounded on the way: a scale block takes the scale of
    its largest value (a power of two, at least 2^-40 and at most 2^40); when a louder token joins it the scale grows
    and what it held is rounded again; a token in its first slot starts it afresh.  See include/nvattn.h."""
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    if _is_fp8(k_cache, k_scale, v_scale):
        _store_kvcache_fp8(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
        return
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    _need_cuda(key, value, k_cache, v_cache, slot_mapping)
    assert key.dtype == value.dtype == k_cache.dtype == v_cache.dtype
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous()
    num_slots = k_cache.numel() // D
    _lib.check(_lib.load().nva_store_kvcache(
        key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
        num_slots, slot_mapping.data_ptr(), N, num_heads, head_dim, key.element_size(), _stream()),
        "store_kvcache")


def _store_kvcache_fp8(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale) -> None:
    N, num_heads, head_dim = key.shape
    G = _scale_block(k_cache, v_cache, k_scale, v_scale)
    NB, BS, KVH, D = k_cache.shape
    assert value.shape == key.shape and (KVH, D) == (num_heads, head_dim)
    assert key.dtype == value.dtype == torch.bfloat16
    if N > 0:
        assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert slot_mapping.numel() == N and slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous()
    _need_cuda(key, value, k_cache, v_cache, slot_mapping)
    assert key.device == value.device == slot_mapping.device == k_cache.device
    with _on(key.device):
        _lib.check(_lib.load().nva_store_kvcache_fp8(
            key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), NB, BS, G, slot_mapping.data_ptr(), N, num_heads, head_dim,
            _stream()), "store_kvcache (8-bit cache)")


def flash_attn_with_kvcache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_seqlens: torch.Tensor,
                            block_table: torch.Tensor, softmax_scale: float, causal: bool = True,
                            out: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                            v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode / verify attention.  q [B, n, H, D] bf16; k_cache/v_cache [NB, BS, KVH, D]; cache_seqlens
    [B] int32 (including the n new tokens); block_table [B, W] int32.  Causal, bottom-right aligned.  With k_scale /
    v_scale the cache is float8_e4m3fn (q and the output stay bf16)."""
    assert causal, "nano-vllm always calls with causal=True"
    if _is_fp8(k_cache, k_scale, v_scale):
        return _decode_fp8(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale, out)
    B, n, H, D = q.shape
    NB, BS, KVH, _ = k_cache.shape
    _need_cuda(q, k_cache, v_cache, cache_seqlens, block_table)
    assert q.dtype == k_cache.dtype == v_cache.dtype == torch.bfloat16
    assert q.stride(-1) == 1 and q.stride(2) == D and q.stride(0) == n * q.stride(1)
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.is_contiguous() and cache_seqlens.numel() == B
    assert block_table.dtype == torch.int32 and block_table.stride(-1) == 1 and block_table.shape[0] == B
    if out is None:
        out = torch.empty(B, n, H, D, dtype=q.dtype, device=q.device)
    else:   # rows are addressed as (b * n + i) * out.stride(1): the same layout rules as q
        _need_cuda(out)
        assert out.dtype == q.dtype and out.shape == q.shape and out.device == q.device
        assert out.stride(-1) == 1 and out.stride(2) == D and out.stride(0) == n * out.stride(1)
    lib = _lib.load()
    ws_bytes = lib.nva_paged_decode_workspace_bytes(B, n, H, KVH, D)
    if ws_bytes == 0:
        raise _lib.NvattnError(f"paged decode does not support q_per_seq={n} with {H // KVH} q heads per kv head")
    with _CALL:
        ws = _workspace(ws_bytes, q.device)
        _lib.check(lib.nva_paged_decode(
            q.data_ptr(), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), NB, BS, cache_seqlens.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), B, n, H, KVH, D, float(softmax_scale), out.data_ptr(),
            out.stride(1), ws.data_ptr(), ws_bytes, _stream()), "paged decode")
    return out


def _decode_fp8(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale, out):
    B, n, H, D = q.shape
    G = _scale_block(k_cache, v_cache, k_scale, v_scale)
    NB, BS, KVH, Dc = k_cache.shape
    _need_cuda(q, k_cache, v_cache, cache_seqlens, block_table)
    assert q.dtype == torch.bfloat16 and Dc == D and H % KVH == 0
    assert q.stride(-1) == 1 and q.stride(2) == D and q.stride(0) == n * q.stride(1)
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.is_contiguous() and cache_seqlens.numel() == B
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    assert block_table.stride(-1) == 1 or block_table.shape[1] == 1
    assert q.device == k_cache.device == cache_seqlens.device == block_table.device
    if out is None:
        out = torch.empty(B, n, H, D, dtype=q.dtype, device=q.device)
    else:   # rows are addressed as (b * n + i) * out.stride(1): the same layout rules as q
        _need_cuda(out)
        assert out.dtype == q.dtype and out.shape == q.shape and out.device == q.device
        assert out.stride(-1) == 1 and out.stride(2) == D and out.stride(0) == n * out.stride(1)
    lib = _lib.load()
    with _on(q.device):
        ws_bytes = lib.nva_paged_attention_fp8_workspace_bytes(n, H, KVH, D)
        if ws_bytes == 0:
            raise _lib.NvattnError(f"paged decode over an 8-bit cache does not support {H // KVH} q heads per kv head "
                                   f"with head_dim {D}")
        with _CALL:
            ws = _workspace(ws_bytes, q.device)
            _lib.check(lib.nva_paged_decode_fp8(
                q.data_ptr(), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), NB, BS, G, cache_seqlens.data_ptr(), block_table.data_ptr(),
                _row_stride(block_table), block_table.shape[1], B, n, H, KVH, D, float(softmax_scale), out.data_ptr(),
                out.stride(1), ws.data_ptr(), ws_bytes, _stream()), "paged decode (8-bit cache)")
    return out


def _varlen_fp8(q, k_cache, v_cache, k_scale, v_scale, max_seqlen_q, cu_seqlens_q, cu_seqlens_k, block_table,
                softmax_scale, out):
    Tq, H, D = q.shape
    G = _scale_block(k_cache, v_cache, k_scale, v_scale)
    NB, BS, KVH, Dc = k_cache.shape
    _need_cuda(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, block_table)
    B = cu_seqlens_q.numel() - 1
    assert q.dtype == torch.bfloat16 and Dc == D and H % KVH == 0
    assert q.stride(-1) == 1 and q.stride(1) == D
    assert cu_seqlens_q.dtype == cu_seqlens_k.dtype == torch.int32 and cu_seqlens_k.numel() == B + 1
    assert cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous()
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] >= B
    assert block_table.stride(-1) == 1 or block_table.shape[1] == 1
    assert q.device == k_cache.device == cu_seqlens_q.device == cu_seqlens_k.device == block_table.device
    if out is None:
        out = torch.empty(Tq, H, D, dtype=q.dtype, device=q.device)
    else:
        _need_cuda(out)
        assert out.dtype == q.dtype and out.shape == q.shape and out.device == q.device
        assert out.stride(-1) == 1 and out.stride(1) == D
    lib = _lib.load()
    with _on(q.device):
        ws_bytes = lib.nva_paged_attention_fp8_workspace_bytes(int(max_seqlen_q), H, KVH, D)
        if ws_bytes == 0:
            raise _lib.NvattnError(f"varlen attention over an 8-bit cache does not support {H // KVH} q heads per kv "
                                   f"head with head_dim {D}")
        with _CALL:
            ws = _workspace(ws_bytes, q.device)
            _lib.check(lib.nva_varlen_attention_fp8(
                q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), NB, BS, G, cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), B, Tq,
                int(max_seqlen_q), block_table.data_ptr(), _row_stride(block_table), block_table.shape[1], H, KVH, D,
                float(softmax_scale), out.data_ptr(), out.stride(0), ws.data_ptr(), ws_bytes, _stream()),
                "varlen attention (8-bit cache)")
    return out


def flash_attn_varlen_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, max_seqlen_q: int,
                           cu_seqlens_q: torch.Tensor, max_seqlen_k: int, cu_seqlens_k: torch.Tensor,
                           softmax_scale: float, causal: bool = True, block_table: torch.Tensor | None = None,
                           out: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                           v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen causal attention.  q [Tq, H, D]; with block_table, k/v are the paged caches [NB, BS, KVH, D],
    else contiguous [Tk, KVH, D] rows (any row stride).  max_seqlen_* are upper bounds only.  With k_scale / v_scale
    (and a block_table) the cache is float8_e4m3fn (q and the output stay bf16)."""
    assert causal, "nano-vllm always calls with causal=True"
    if _is_fp8(k, k_scale, v_scale):
        assert block_table is not None, "an 8-bit cache is read through a block_table"
        return _varlen_fp8(q, k, v, k_scale, v_scale, max_seqlen_q, cu_seqlens_q, cu_seqlens_k, block_table,
                           softmax_scale, out)
    Tq, H, D = q.shape
    _need_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, block_table)
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16
    assert q.stride(-1) == 1 and q.stride(1) == D
    assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32
    assert cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous()
    B = cu_seqlens_q.numel() - 1
    if out is None:
        out = torch.empty(Tq, H, D, dtype=q.dtype, device=q.device)
    else:
        _need_cuda(out)
        assert out.dtype == q.dtype and out.shape == q.shape and out.device == q.device
        assert out.stride(-1) == 1 and out.stride(1) == D
    lib = _lib.load()
    if block_table is not None:
        NB, BS, KVH, _ = k.shape
        assert k.is_contiguous() and v.is_contiguous()
        assert block_table.dtype == torch.int32 and block_table.stride(-1) == 1
        kp, kst, vp, vst, Tk = 0, 0, 0, 0, 0
        kc, vc, bt, bts = k.data_ptr(), v.data_ptr(), block_table.data_ptr(), block_table.stride(0)
    else:
        Tk, KVH, _ = k.shape
        assert k.stride(-1) == 1 and k.stride(1) == D and v.stride(-1) == 1 and v.stride(1) == D
        NB, BS = 0, 0
        kp, kst, vp, vst = k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0)
        kc, vc, bt, bts = 0, 0, 0, 0
    ws_bytes = lib.nva_varlen_workspace_bytes(B, Tq, H, KVH, D)
    with _CALL:
        ws = _workspace(ws_bytes, q.device)
        _lib.check(lib.nva_varlen_attention(
            q.data_ptr(), q.stride(0), kp, kst, vp, vst, kc, vc, NB, BS, cu_seqlens_q.data_ptr(),
            cu_seqlens_k.data_ptr(), B, Tq, Tk, int(max_seqlen_q), int(max_seqlen_k), bt, bts, H, KVH, D,
            float(softmax_scale), out.data_ptr(), out.stride(0), ws.data_ptr(), ws_bytes, _stream()),
            "varlen attention")
    return out


def greedy_accept(target_ids: torch.Tensor, draft_ids: torch.Tensor, num_drafts: torch.Tensor):
    """Integer greedy accept length: target [S, K+1], drafts [S, K], num_drafts [S] (all int32 or all int64).
    Returns (num_accepted [S], next_token [S]) in the same dtype."""
    _need_cuda(target_ids, draft_ids, num_drafts)
    S, K1 = target_ids.shape
    K = K1 - 1
    dt = target_ids.dtype
    assert dt in (torch.int32, torch.int64) and draft_ids.dtype == dt and num_drafts.dtype == dt
    assert target_ids.stride(-1) == 1 and num_drafts.is_contiguous() and num_drafts.numel() == S
    assert draft_ids.shape == (S, K) and (K == 0 or draft_ids.stride(-1) == 1)
    acc = torch.empty(S, dtype=dt, device=target_ids.device)
    nxt = torch.empty(S, dtype=dt, device=target_ids.device)
    _lib.check(_lib.load().nva_greedy_accept(
        target_ids.data_ptr(), target_ids.stride(0), draft_ids.data_ptr() if K else 0, draft_ids.stride(0) if K else 0,
        num_drafts.data_ptr(), S, K, target_ids.element_size(), acc.data_ptr(), nxt.data_ptr(), _stream()),
        "greedy accept")
    return acc, nxt


def shard_argmax(logits: torch.Tensor, vocab_offset: int = 0) -> torch.Tensor:
    """Per-row argmax keys of one vocabulary shard of logits [rows, V_shard] (bf16 or float32, unit column stride):
    int64 [rows] holding orderable(max) << 32 | (0xFFFFFFFF - (vocab_offset + first index of the max)) as raw bits.
    The largest key of a row over all shards (compared as unsigned) is the row's argmax with torch's tie rule; see
    shard_accept.  Replaces the per-rank part of the logits gather + argmax (embed_head.py:56-68, sampler.py:66)."""
    _need_cuda(logits)
    assert logits.dim() == 2 and logits.stride(-1) == 1
    assert logits.dtype in (torch.bfloat16, torch.float32)
    rows, vocab = logits.shape
    keys = torch.empty(rows, dtype=torch.int64, device=logits.device)
    _lib.check(_lib.load().nva_shard_argmax(logits.data_ptr(), logits.stride(0), rows, vocab, int(vocab_offset),
                                            logits.element_size(), keys.data_ptr(), _stream()), "shard argmax")
    return keys


def shard_accept(keys: torch.Tensor, draft_ids: torch.Tensor, num_drafts: torch.Tensor):
    """Greedy accept from argmax keys: keys [num_shards, S, K+1] (int64 raw bits from shard_argmax of each shard,
    contiguous), draft_ids [S, K], num_drafts [S] (int32 or int64, same dtype).  Returns (num_accepted [S],
    next_token [S]) in that dtype: verify_drafts' greedy result (sampler.py:66-82) on the concatenated shards."""
    _need_cuda(keys, draft_ids, num_drafts)
    num_shards, S, K1 = keys.shape
    K = K1 - 1
    dt = draft_ids.dtype
    assert keys.dtype == torch.int64 and keys.is_contiguous()
    assert dt in (torch.int32, torch.int64) and num_drafts.dtype == dt
    assert num_drafts.is_contiguous() and num_drafts.numel() == S
    assert draft_ids.shape == (S, K) and (K == 0 or draft_ids.stride(-1) == 1)
    acc = torch.empty(S, dtype=dt, device=keys.device)
    nxt = torch.empty(S, dtype=dt, device=keys.device)
    _lib.check(_lib.load().nva_shard_accept(
        keys.data_ptr(), num_shards, S, K, draft_ids.data_ptr() if K else 0, draft_ids.stride(0) if K else 0,
        num_drafts.data_ptr(), draft_ids.element_size(), acc.data_ptr(), nxt.data_ptr(), _stream()), "shard accept")
    return acc, nxt


def _settings(rows: int, device, temperatures, top_k, top_p, min_p):
    """Checks the per-row sampling settings; returns their pointers (0: off)."""
    shape, out = (rows,), []
    for x, dt in ((temperatures, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32)):
        if x is None:
            out.append(0)
            continue
        assert x.dtype is dt and x.shape == shape and x.is_contiguous() and x.device == device
        out.append(x.data_ptr())
    return out


def sample_tokens(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits [R, V] (bf16 or float32, unit column stride), int64 [R], from the uniform numbers
    uniforms [R] in [0, 1) (float32 or float64).  temperatures [R] float32 (<= 0: argmax), top_k [R] int32 (<= 0: off),
    top_p [R] float32 (>= 1: off), min_p [R] float32 (<= 0: off).  The rules are in include/nvattn.h."""
    _need_cuda(logits, temperatures, uniforms, top_k, top_p, min_p)
    assert logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32)
    R, V = logits.shape
    assert logits.stride(1) == 1 or V == 1
    assert uniforms.dtype in (torch.float32, torch.float64) and uniforms.shape == (R,) and uniforms.is_contiguous()
    assert temperatures is not None and uniforms.device == logits.device
    t, k, p, m = _settings(R, logits.device, temperatures, top_k, top_p, min_p)
    ids = torch.empty(R, dtype=torch.int64, device=logits.device)
    lib = _lib.load()
    ws, ws_bytes = None, 0
    if not (k or p or m):
        ws_bytes = lib.nva_sample_workspace_bytes(R, V, logits.element_size())
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device)
    with _on(logits.device):
        _lib.check(lib.nva_sample_tokens(
            logits.data_ptr(), _row_stride(logits), R, V, logits.element_size(), t,
            k, p, m, uniforms.data_ptr(), uniforms.element_size(), ids.data_ptr(), ws.data_ptr() if ws_bytes else 0,
            ws_bytes, _stream()), "sample tokens")
    return ids


def verify_sampled(logits: torch.Tensor, draft_ids: torch.Tensor, num_drafts: torch.Tensor,
                   temperatures: torch.Tensor, accept_uniforms: torch.Tensor, uniforms: torch.Tensor,
                   top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                   min_p: torch.Tensor | None = None):
    """Speculative sampling of fixed drafts: logits [S * (K+1), V], draft_ids [S, K] and num_drafts [S] (both int32 or
    both int64), settings and uniforms [S] per sequence, accept_uniforms [S, K] (the uniforms' dtype).  Returns
    (num_accepted [S], next_token [S]) in the ids' dtype.  The rules are in include/nvattn.h."""
    _need_cuda(logits, draft_ids, num_drafts, temperatures, accept_uniforms, uniforms, top_k, top_p, min_p)
    S, K = draft_ids.shape
    dt, dev = draft_ids.dtype, logits.device
    assert logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32)
    rows, V = logits.shape
    assert rows == S * (K + 1) and (logits.stride(1) == 1 or V == 1)
    assert dt in (torch.int32, torch.int64) and num_drafts.dtype == dt
    assert num_drafts.shape == (S,) and num_drafts.is_contiguous()
    assert K <= 1 or (draft_ids.stride(1) == 1 and accept_uniforms.stride(1) == 1)
    assert uniforms.dtype in (torch.float32, torch.float64) and uniforms.shape == (S,) and uniforms.is_contiguous()
    assert accept_uniforms.dtype == uniforms.dtype and accept_uniforms.shape == (S, K)
    assert temperatures is not None
    assert dev == draft_ids.device == num_drafts.device == accept_uniforms.device == uniforms.device
    t, k, p, m = _settings(S, dev, temperatures, top_k, top_p, min_p)
    acc, nxt = torch.empty_like(num_drafts), torch.empty_like(num_drafts)
    lib = _lib.load()
    ws_bytes = 16 * rows if k or p or m else lib.nva_sample_workspace_bytes(rows, V, logits.element_size())
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.check(lib.nva_verify_sampled(
            logits.data_ptr(), _row_stride(logits), S, K, V, logits.element_size(),
            draft_ids.data_ptr() if K else 0, _row_stride(draft_ids) if K else 0, num_drafts.data_ptr(),
            draft_ids.element_size(), t, k, p, m, accept_uniforms.data_ptr() if K else 0,
            _row_stride(accept_uniforms) if K else 0, uniforms.data_ptr(), uniforms.element_size(),
            acc.data_ptr(), nxt.data_ptr(), ws.data_ptr(), ws_bytes, _stream()), "verify sampled")
    return acc, nxt


def qk_norm_rope_store(qkv: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                       q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float, num_heads: int,
                       num_kv_heads: int, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                       slot_mapping: torch.Tensor | None = None, want_k: bool = False):
    """Qwen3's attention prologue in one kernel: from the fused projection output qkv [T, (H + 2 KVH) * 128], the
    normalised and rotated q [T, H, 128] (returned), the same for k (returned when want_k, else None), and, with a
    cache, k and v scattered to slot_mapping's slots (qwen3.py:88-97 then attention.py:61-62).  cos_sin_cache is the
    reference RotaryEmbedding's [max_position, 1 or none, 128] float32 table.  Returns (q, k, v) with v a view of
    qkv, as Qwen3Attention.pre_attn returns them."""
    _need_cuda(qkv, positions, cos_sin_cache, q_norm_weight, k_norm_weight)
    D = 128
    T = qkv.shape[0]
    assert qkv.dim() == 2 and qkv.shape[1] == (num_heads + 2 * num_kv_heads) * D and qkv.stride(1) == 1
    assert qkv.dtype == torch.bfloat16 and q_norm_weight.dtype == k_norm_weight.dtype == torch.bfloat16
    assert positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == T
    table = cos_sin_cache.reshape(-1, D)
    assert table.dtype == torch.float32 and table.is_contiguous()
    q = torch.empty(T, num_heads, D, dtype=qkv.dtype, device=qkv.device)
    k = torch.empty(T, num_kv_heads, D, dtype=qkv.dtype, device=qkv.device) if want_k else None
    if slot_mapping is not None:
        _need_cuda(k_cache, v_cache, slot_mapping)
        assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous() and slot_mapping.numel() == T
        assert k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.dtype == qkv.dtype
        assert k_cache.stride(1) == num_kv_heads * D
        num_slots = k_cache.numel() // (num_kv_heads * D)
    else:
        num_slots = 0
    _lib.check(_lib.load().nva_qk_norm_rope_store(
        qkv.data_ptr(), qkv.stride(0), T, num_heads, num_kv_heads, D, positions.data_ptr(), table.data_ptr(),
        table.shape[0], q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps), q.data_ptr(), q.stride(0),
        k.data_ptr() if k is not None else 0, k.stride(0) if k is not None else 0,
        k_cache.data_ptr() if slot_mapping is not None else 0, v_cache.data_ptr() if slot_mapping is not None else 0,
        num_slots, slot_mapping.data_ptr() if slot_mapping is not None else 0, _stream()), "qk norm rope store")
    v = qkv[:, (num_heads + num_kv_heads) * D:].view(T, num_kv_heads, D)
    return q, k, v
