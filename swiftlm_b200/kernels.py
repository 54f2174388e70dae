"""Host-side mirror of the reference's kernel entry points (`public enum DFlashKernels`,
Sources/DFlash/DFlashKernels.swift of the SwiftLM tree) on top of the C ABI.

Same names (snake_case), argument meaning, layouts and error behaviour as the Swift API:
inputs are never mutated, outputs are fresh tensors, `batched_sdpa_2pass` returns None for
shapes outside the supported set exactly where the reference returns nil.  torch is used only
for device memory and streams; every computation happens in libdflash_cuda.so.  There is no
CPU path: tensors must live on a CUDA device.
"""
from __future__ import annotations

from typing import Optional, Tuple

import ctypes as C
import functools

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16,
       torch.uint8: _lib.U8, torch.bool: _lib.U8}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("DFlash kernels run on a CUDA device only (no CPU fallback)")


def _mask_arg(mask: Optional[torch.Tensor]):
    if mask is None:
        return None, 0
    if mask.dtype not in _DT:
        mask = mask.to(torch.float32)
    return mask.contiguous(), _DT[mask.dtype]


def _n_arg(n_per_seq, B, device):
    if n_per_seq is None:
        return None
    n = torch.as_tensor(n_per_seq, device=device).to(torch.int32).contiguous()
    if n.numel() != B:
        raise ValueError("n_per_seq must have one entry per sequence")
    return n


def gated_delta_kernel_with_tape(q, k, v, g, beta, state, mask=None, n_per_seq=None,
                                 want_tape: bool = True) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """DFlashKernels.gatedDeltaKernelWithTape (Sources/DFlash/DFlashKernels.swift:316-324).

    q,k [B,T,Hk,Dk]; v [B,T,Hv,Dv]; g [B,T,Hv] or [B,T,Hv,Dk]; beta [B,T,Hv];
    state [B,Hv,Dv,Dk] (kept in fp32); mask [B,T] optional.  Returns (y [B,T,Hv,Dv] in q's
    dtype, new state fp32, innovation tape fp32 [B,T,Hv,Dv]).
    n_per_seq (int32 [B], not in the reference signature) runs only the first n steps of each
    sequence: this is the replay of a recorded block to its accepted length.
    """
    _need_cuda(q, k, v, g, beta, state)
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    dt = q.dtype
    if dt not in (torch.float32, torch.bfloat16, torch.float16):
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, f"input dtype {dt}")
    q, k, v, g, beta = (x.to(dt).contiguous() for x in (q, k, v, g, beta))
    state = state.to(torch.float32).contiguous()
    mask, mdt = _mask_arg(mask)
    n = _n_arg(n_per_seq, B, q.device)
    y = torch.empty((B, T, Hv, Dv), dtype=dt, device=q.device)
    state_out = torch.empty_like(state)
    tape = torch.empty((B, T, Hv, Dv), dtype=torch.float32, device=q.device) if want_tape else None
    _lib.check(_lib.lib().dflash_gated_delta_tape(
        _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(mask), _ptr(n),
        _ptr(y), _ptr(state_out), _ptr(tape), B, T, Hk, Hv, Dk, Dv, int(g.dim() == 4), _DT[dt], mdt,
        _stream()))
    return y, state_out, tape


def tape_replay_kernel(tape, k, g, state, mask=None, n_per_seq=None) -> torch.Tensor:
    """DFlashKernels.tapeReplayKernel (Sources/DFlash/DFlashKernels.swift:252-258).

    tape [B,T,Hv,Dv] (fp32), k [B,T,Hk,Dk], g [B,T,Hv] or [B,T,Hv,Dk], state [B,Hv,Dv,Dk].
    Returns the replayed state.  n_per_seq replays only the first n steps per sequence (what
    the reference's caller does by slicing, Sources/DFlash/RecurrentRollbackCache.swift:115-118).
    """
    _need_cuda(tape, k, g, state)
    B, T, Hv, Dv = tape.shape
    Hk, Dk = k.shape[2], k.shape[3]
    dt = k.dtype
    if dt not in (torch.float32, torch.bfloat16, torch.float16):
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, f"input dtype {dt}")
    tape = tape.to(torch.float32).contiguous()
    k = k.contiguous()
    g = g.to(dt).contiguous()
    state = state.to(torch.float32).contiguous()
    mask, mdt = _mask_arg(mask)
    n = _n_arg(n_per_seq, B, k.device)
    out = torch.empty_like(state)
    _lib.check(_lib.lib().dflash_tape_replay(
        _ptr(tape), _ptr(k), _ptr(g), _ptr(state), _ptr(mask), _ptr(n), _ptr(out),
        B, T, Hk, Hv, Dk, Dv, int(g.dim() == 4), _DT[dt], mdt, _stream()))
    return out


_workspaces = {}


def _workspace(device, nbytes: int) -> Optional[torch.Tensor]:
    if nbytes == 0:
        return None
    key = (device.index, torch.cuda.current_stream().cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def batched_sdpa_2pass(queries, keys, values, scale: float, mask=None, kv_len=None,
                       page_table=None, out=None, n_max=None) -> Optional[torch.Tensor]:
    """DFlashKernels.batchedSDPA2Pass (Sources/DFlash/DFlashKernels.swift:737-743).

    queries [B,Hq,16,D]; keys/values [B,Hkv,N,D] (or, with page_table int32 [B,max_pages],
    page pools [num_pages,Hkv,page_tokens,D]); optional additive mask [B,Hq,16,N].
    Returns [B,Hq,16,D] in the input dtype, or None where the reference returns nil
    (query length != 16, dtype not bf16/f16, head_dim not in {128,256}, Hq % Hkv != 0).
    """
    _need_cuda(queries, keys, values)
    if queries.dim() != 4 or keys.dim() != 4 or values.dim() != 4:
        return None
    B, Hq, T, D = queries.shape
    dt = queries.dtype
    if T != 16 or dt not in (torch.bfloat16, torch.float16):
        return None
    if D not in (128, 256) or values.shape[3] != D:
        return None
    Hkv = keys.shape[1]
    if Hkv <= 0 or Hq % Hkv != 0:
        return None
    q = queries.contiguous()
    k = keys.to(dt).contiguous()
    v = values.to(dt).contiguous()
    if kv_len is not None:
        kv_len = torch.as_tensor(kv_len, device=q.device).to(torch.int32).contiguous()
    if page_table is None:
        N, page_tokens, max_pages, num_pages = keys.shape[2], 0, 0, 0
    else:
        if kv_len is None:
            raise ValueError("paged KV needs kv_len")
        page_table = page_table.to(torch.int32).contiguous()
        page_tokens, max_pages, num_pages = keys.shape[2], page_table.shape[1], keys.shape[0]
        # n_max avoids a host read of kv_len on the hot path
        N = int(n_max) if n_max is not None else int(kv_len.max())
    if mask is not None:
        mask = mask.to(dt).expand(B, Hq, 16, N).contiguous()
    if out is None:
        out = torch.empty_like(q)
    L = _lib.lib()
    ws = _workspace(q.device, L.dflash_verify_sdpa_workspace_bytes(B, Hq, Hkv, D, N))
    try:
        _lib.check(L.dflash_verify_sdpa(
            _ptr(q), _ptr(k), _ptr(v), _ptr(page_table), _ptr(kv_len), _ptr(mask), _ptr(out),
            _ptr(ws), 0 if ws is None else ws.numel(), B, Hq, Hkv, T, D, N, page_tokens, max_pages,
            num_pages, float(scale), _DT[dt], _lib.KV_DENSE, _stream()))
    except _lib.DFlashUnsupported:
        return None
    return out


def greedy_tokens_with_mask(logits: torch.Tensor, suppress_token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """DFlashRuntime.greedyTokensWithMask (Sources/DFlash/DFlashRuntime.swift:118-128).
    logits [..., V]; returns token ids (uint32 values held in an int64-free int32 view)."""
    _need_cuda(logits)
    V = logits.shape[-1]
    flat = logits.contiguous().view(-1, V)
    sup = None
    if suppress_token_mask is not None:
        sup = suppress_token_mask.to(device=logits.device, dtype=torch.uint8).contiguous()
    post = torch.empty(flat.shape[0], dtype=torch.int32, device=logits.device)
    _lib.check(_lib.lib().dflash_greedy_tokens(_ptr(flat), _ptr(sup), _ptr(post), flat.shape[0], V,
                                              _DT[logits.dtype], _stream()))
    return post.view(logits.shape[:-1])


def accept_lengths(posterior: torch.Tensor, verify_ids: torch.Tensor):
    """DFlashRuntime.matchAcceptanceLength + the commit arithmetic
    (Sources/DFlash/DFlashRuntime.swift:133-142, :523-547), batched over sequences.
    posterior, verify_ids int32 [B,T].  Returns (accept [B], next_token [B], replay_len [B])."""
    _need_cuda(posterior, verify_ids)
    B, T = verify_ids.shape
    posterior = posterior.to(torch.int32).contiguous()
    verify_ids = verify_ids.to(torch.int32).contiguous()
    acc = torch.empty(B, dtype=torch.int32, device=posterior.device)
    nxt = torch.empty_like(acc)
    rep = torch.empty_like(acc)
    _lib.check(_lib.lib().dflash_accept_lengths(_ptr(posterior), _ptr(verify_ids), _ptr(acc), _ptr(nxt),
                                               _ptr(rep), B, T, _stream()))
    return acc, nxt, rep


def gather_logits_rows(logits: torch.Tensor, row_per_seq: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [B,T,V], row_per_seq int32 [B] (the accepted count) -> [B,V]: each sequence's logits row at its accepted
    position, the row whose argmax is the next staged token (Sources/DFlash/DFlashRuntime.swift:547)."""
    _need_cuda(logits, row_per_seq)
    B, T, V = logits.shape
    logits = logits.contiguous()
    if out is None:
        out = torch.empty(B, V, dtype=logits.dtype, device=logits.device)
    _lib.check(_lib.lib().dflash_gather_logits_rows(_ptr(logits), _ptr(row_per_seq.to(torch.int32).contiguous()), _ptr(out),
                                                   B, T, V, _DT[logits.dtype], _stream()))
    return out


def turbo_decode_into(packed, signs, norm, rnorm, out: torch.Tensor) -> None:
    """turbo_decode into a caller-owned tensor (any shape holding norm.numel() * 128 values)."""
    _need_cuda(packed, norm, out)
    n = norm.numel()
    if out.numel() != n * 128 or not out.is_contiguous():
        raise _lib.DFlashError(_lib.ERR_INVALID_ARG, "turbo_decode_into: out must be contiguous with 128 values per block")
    _lib.check(_lib.lib().dflash_turbo_decode(_ptr(packed.contiguous()), _ptr(signs), _ptr(norm.contiguous()),
                                             _ptr(rnorm), _ptr(out), n, int(signs is not None), _DT[out.dtype], _stream()))


def device_status() -> None:
    """Raises if a kernel's bounded device-side wait gave up since the last check."""
    _lib.check(_lib.lib().dflash_device_status(_stream()))


def launch_count() -> int:
    return int(_lib.lib().dflash_launch_count())


def tape_replay_into(tape, k, g, state, n_per_seq, state_out, mask=None) -> None:
    """Allocation-free form of tape_replay_kernel: every buffer is supplied by the caller (contiguous, on the current
    device; tape and state fp32).  state_out may be the same tensor as state."""
    B, T, Hv, Dv = tape.shape
    Hk, Dk = k.shape[2], k.shape[3]
    mask_t, mdt = _mask_arg(mask)
    _lib.check(_lib.lib().dflash_tape_replay(
        _ptr(tape), _ptr(k), _ptr(g), _ptr(state), _ptr(mask_t), _ptr(n_per_seq), _ptr(state_out),
        B, T, Hk, Hv, Dk, Dv, int(g.dim() == 4), _DT[k.dtype], mdt, _stream()))


def kv_append(k_new, v_new, k_cache, v_cache, kv_len=None, len_all: int = 0, page_table=None, kv_len_out=None) -> None:
    """Writes the block's rows k_new / v_new [B,Hkv,T,D] behind the committed tokens of a dense cache [B,Hkv,capacity,D]
    or, with page_table int32[B,max_pages], of a page pool [pages,Hkv,page_tokens,D]: row t of sequence b lands at
    position kv_len[b] + t (len_all + t without kv_len).  kv_len_out receives kv_len + T, the length the verify
    attention sees.  Replaces the cache update before the target forward (Sources/DFlash/DFlashRuntime.swift:188-223)."""
    B, Hkv, T, D = k_new.shape
    if page_table is not None:
        num_pages, page_tokens, max_pages, capacity = k_cache.shape[0], k_cache.shape[2], page_table.shape[1], 0
    else:
        num_pages, page_tokens, max_pages, capacity = 0, 0, 0, k_cache.shape[2]
    _lib.check(_lib.lib().dflash_kv_append(
        _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache), _ptr(page_table), _ptr(kv_len), int(len_all),
        _ptr(kv_len_out), B, Hkv, T, D, capacity, page_tokens, max_pages, num_pages, _DT[k_new.dtype], _stream()))


def kv_commit(kv_len, commit, block: int = 16) -> None:
    """kv_len[b] += clamp(commit[b], 0, block): keeps the accepted prefix of the block just appended and
    leaves the rejected rows to be overwritten (the reference's cache.trim(offset - targetLen))."""
    _lib.check(_lib.lib().dflash_kv_commit(_ptr(kv_len), _ptr(commit), kv_len.numel(), int(block), _stream()))


# ---- the cache outside the verify cycle: plain decoding, prompts, eviction (no counterpart among the reference's kernels) ----

def _bad(what: str):
    return _lib.DFlashError(_lib.ERR_INVALID_ARG, what)


# The calls below are made once a token: what they check and allocate is kept to a few microseconds.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name: str, device_index: int, *sizes) -> int:
    with torch.cuda.device(device_index):
        return getattr(_lib.lib(), name)(*sizes)


def _on_its_device(fn):
    """Runs fn with its first argument's device current: allocation, stream and launch all go to it."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kwargs):
        t = args[0] if args else kwargs.get(first)
        if t is None:
            raise TypeError(f"{fn.__name__}() needs {first}")
        if not t.is_cuda:
            _need_cuda(t)
        if t.device.index == torch.cuda.current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(t.device):
            return fn(*args, **kwargs)
    return call


def _same_device(device, *others):
    for t in others:
        if t is not None and t.device != device:
            raise _bad(f"tensors on different devices: {device} and {t.device}")


def _int_vector(x, n: int, device, name: str):
    if x is None:
        return None
    if not (isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.device == device and x.is_contiguous()):
        x = torch.as_tensor(x, device=device).to(torch.int32).contiguous()
    if x.dim() != 1 or x.shape[0] != n:
        raise _bad(f"{name} must have one entry per sequence")
    return x


def _cache_shape(keys, page_table, n_max, B: int):
    """(page_table as the kernels take it, N, page_tokens, max_pages, num_pages) of a dense cache [B,Hkv,capacity,D] or of a
    page pool [num_pages,Hkv,page_tokens,D]."""
    if page_table is None:
        if keys.shape[0] != B:
            raise _bad("a dense cache has one entry per sequence")
        return None, keys.shape[2], 0, 0, 0
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise _bad("page_table must be [B, max_pages]")
    if page_table.dtype != torch.int32 or not page_table.is_contiguous():
        page_table = page_table.to(torch.int32).contiguous()
    num_pages, _, page_tokens, _ = keys.shape
    max_pages = page_table.shape[1]
    capacity = max_pages * page_tokens
    return page_table, (capacity if n_max is None else min(int(n_max), capacity)), page_tokens, max_pages, num_pages


def _cache_tensors(queries, dims: int, keys, values, *others):
    """What the three attention calls refuse alike."""
    if queries.dim() != dims:
        raise _bad("queries must be " + ("[B, Hq, D]" if dims == 3 else "[B, Hq, T, D]"))
    if keys.dim() != 4 or queries.shape[-1] != keys.shape[3]:
        raise _bad("keys must be 4-dimensional, with the queries' head dimension")
    dt = queries.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, f"dtype {dt} (bf16 or f16)")
    if keys.dtype is not dt or (values is not None and values.dtype is not dt):
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, "queries, keys and values must have one dtype")
    if values is not None and values.shape != keys.shape:
        raise _bad("keys and values must have one shape")
    _same_device(queries.device, keys, values, *others)


def _mass_arg(mass, B: int, Hkv: int, N: int, name: str = "mass"):
    if mass.dtype != torch.float32 or mass.dim() != 3 or mass.shape[:2] != (B, Hkv) or mass.shape[2] < N or not mass.is_contiguous():
        raise _bad(f"{name} must be a contiguous fp32 tensor [B, Hkv, >= {N}]")
    return mass


def _out_arg(out, like: torch.Tensor, name: str = "out"):
    if out is None:
        return torch.empty_like(like)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous():
        raise _bad(f"{name} must be a contiguous tensor of the queries' shape, dtype and device")
    return out


def _scratch(nbytes: int, device) -> Optional[torch.Tensor]:
    """Workspace of one call.  Taken from torch's allocator call by call, so that calls on several streams and calls captured
    into different CUDA graphs never share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


@_on_its_device
def decode_sdpa(queries, keys, values, scale: float, kv_len=None, page_table=None, window: int = 0, sinks: int = 0,
                mass: Optional[torch.Tensor] = None, return_lse: bool = False, out=None, n_max=None):
    """Attention of one new token per sequence over its cache, the new token being the last cached one.

    queries [B,Hq,D]; keys/values a dense cache [B,Hkv,capacity,D] or, with page_table int32 [B,max_pages], page pools
    [num_pages,Hkv,page_tokens,D] (page_tokens a multiple of 16); kv_len int32 [B]: cached tokens (0 for an unused place:
    its output is 0).  window > 0: the last `window` tokens are visible, and the first `sinks`.  mass fp32
    [B,Hkv,>= capacity]: the weight of every visible token, summed over the query heads of its KV head, is added to
    it.  n_max: an upper bound of kv_len for a page pool, when less than the table's reach is in use.  out: a tensor like
    queries, or queries itself.
    Returns [B,Hq,D], or (that, lse fp32 [B,Hq]) with return_lse.
    """
    _cache_tensors(queries, 3, keys, values, page_table, mass, out)
    scale, window, sinks = float(scale), int(window), int(sinks)
    B, Hq, D = queries.shape
    Hkv, device = keys.shape[1], queries.device
    page_table, N, page_tokens, max_pages, num_pages = _cache_shape(keys, page_table, n_max, B)
    stride = 0
    if mass is not None:
        stride = _mass_arg(mass, B, Hkv, N).shape[2]
    q, k, v = queries.contiguous(), keys.contiguous(), values.contiguous()
    kv_len = _int_vector(kv_len, B, device, "kv_len")
    out = _out_arg(out, q)
    lse = torch.empty((B, Hq), dtype=torch.float32, device=device) if return_lse else None
    need = _workspace_bytes("dflash_decode_sdpa_workspace_bytes", device.index, B, Hq, Hkv, D, N, window, sinks, int(mass is not None))
    ws = _scratch(need, device)
    _lib.check(_lib.lib().dflash_decode_sdpa(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(page_table), _ptr(kv_len), out.data_ptr(), _ptr(lse), _ptr(mass), _ptr(ws), need,
        B, Hq, Hkv, D, N, page_tokens, max_pages, num_pages, stride, window, sinks, scale, _DT[q.dtype], _raw_stream(device.index)))
    return (out, lse) if return_lse else out


@_on_its_device
def prompt_sdpa(queries, keys, values, scale: float, q_len=None, kv_len=None, page_table=None, window: int = 0, sinks: int = 0,
                return_lse: bool = False, out=None, n_max=None):
    """Attention of a prompt, or of a chunk of one behind what the cache holds already, with the chunk's own rows in the
    cache (append first).

    queries [B,Hq,T,D]; keys/values, kv_len, page_table, window, sinks, n_max as for decode_sdpa.  q_len int32 [B]: query
    rows in use (default T); row r of sequence b stands at position kv_len[b] - q_len[b] + r and sees the tokens up to its
    own, within the window or among the sinks.  Rows at and behind q_len[b] are left as they are in `out`.
    Returns [B,Hq,T,D], or (that, lse fp32 [B,Hq,T]) with return_lse (-inf on rows that see nothing or are not in use).
    """
    _cache_tensors(queries, 4, keys, values, page_table, out)
    scale, window, sinks = float(scale), int(window), int(sinks)
    B, Hq, T, D = queries.shape
    Hkv, device = keys.shape[1], queries.device
    page_table, N, page_tokens, max_pages, num_pages = _cache_shape(keys, page_table, n_max, B)
    q, k, v = queries.contiguous(), keys.contiguous(), values.contiguous()
    kv_len, q_len = _int_vector(kv_len, B, device, "kv_len"), _int_vector(q_len, B, device, "q_len")
    out = _out_arg(out, q)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=device) if return_lse else None
    need = _workspace_bytes("dflash_prompt_sdpa_workspace_bytes", device.index, B, Hq, Hkv, T, D, N)
    ws = _scratch(need, device)
    _lib.check(_lib.lib().dflash_prompt_sdpa(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(page_table), _ptr(q_len), _ptr(kv_len), out.data_ptr(), _ptr(lse), _ptr(ws), need,
        B, Hq, Hkv, T, D, N, page_tokens, max_pages, num_pages, window, sinks, scale, _DT[q.dtype], _raw_stream(device.index)))
    return (out, lse) if return_lse else out


@_on_its_device
def attention_mass(queries, keys, lse, scale: float, mass, q_len=None, kv_len=None, page_table=None, window: int = 0,
                   sinks: int = 0, n_max=None) -> None:
    """Adds to mass fp32 [B,Hkv,>= capacity] the weight that the queries [B,Hq,T,D] give to every cached token, summed over
    rows and the query heads of a KV head: exp(scale * q.k - lse) with the lse [B,Hq,T] of prompt_sdpa over the same cache
    (all of a chunk's rows, or its last ones: the rows given are the last T, or q_len, tokens of the cache)."""
    _cache_tensors(queries, 4, keys, None, page_table, lse, mass)
    scale, window, sinks = float(scale), int(window), int(sinks)
    B, Hq, T, D = queries.shape
    Hkv, device = keys.shape[1], queries.device
    if lse.dtype != torch.float32 or lse.shape != (B, Hq, T):
        raise _bad("lse must be fp32 [B, Hq, T]")
    page_table, N, page_tokens, max_pages, num_pages = _cache_shape(keys, page_table, n_max, B)
    _mass_arg(mass, B, Hkv, N)
    q, k, lse = queries.contiguous(), keys.contiguous(), lse.contiguous()
    kv_len, q_len = _int_vector(kv_len, B, device, "kv_len"), _int_vector(q_len, B, device, "q_len")
    need = _workspace_bytes("dflash_attention_mass_workspace_bytes", device.index, B, Hq, Hkv, T, D, N)
    ws = _scratch(need, device)
    _lib.check(_lib.lib().dflash_attention_mass(
        q.data_ptr(), k.data_ptr(), _ptr(page_table), _ptr(q_len), _ptr(kv_len), lse.data_ptr(), mass.data_ptr(), _ptr(ws), need,
        B, Hq, Hkv, T, D, N, page_tokens, max_pages, num_pages, mass.shape[2], window, sinks, scale, _DT[q.dtype],
        _raw_stream(device.index)))


@_on_its_device
def kv_evict(k_cache, v_cache, mass, kv_len, budget: int, recent: int, sinks: int = 0, page_table=None, kv_len_out=None,
             mass_out=None, kept=None, n_max=None) -> torch.Tensor:
    """Cuts every sequence longer than `budget` tokens down to it, per KV head and in place: the first `sinks` tokens, the
    last `recent` and the heaviest of the others (mass fp32 [B,Hkv,>= capacity], ties to the lowest index) move to the
    front of the cache in the order they are in.

    k_cache/v_cache a dense cache [B,Hkv,capacity,D] or, with page_table, page pools; the pages of a sequence that is cut
    belong to it alone.  mass_out (default: mass itself) receives the masses of the rows that stay and zeros up to the
    old length; kept int32 [B,Hkv,budget], if given, their old places (-1 behind the last).  Returns kv_len_out
    (default: kv_len itself, updated): min(kv_len, budget).
    """
    _need_cuda(mass, kv_len)
    device = k_cache.device
    _same_device(device, v_cache, mass, kv_len, page_table, kv_len_out, mass_out, kept)
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise _bad("k_cache and v_cache must be two 4-dimensional tensors of one shape and dtype")
    if k_cache.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, f"dtype {k_cache.dtype}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise _bad("the caches are changed in place and must be contiguous")
    B, Hkv, D = kv_len.numel(), k_cache.shape[1], k_cache.shape[3]
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    page_table, N, page_tokens, max_pages, num_pages = _cache_shape(k_cache, page_table, n_max, B)
    kv_len_out = kv_len if kv_len_out is None else kv_len_out
    for t, name in ((kv_len, "kv_len"), (kv_len_out, "kv_len_out")):
        if t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous():
            raise _bad(f"{name} must be a contiguous int32 tensor [B]")
    mass_out = mass if mass_out is None else mass_out
    _mass_arg(mass, B, Hkv, N)
    _mass_arg(mass_out, B, Hkv, N, "mass_out")
    if mass_out.shape != mass.shape:
        raise _bad("mass_out must have the shape of mass")
    if kept is not None and (kept.dtype != torch.int32 or kept.shape != (B, Hkv, budget) or not kept.is_contiguous()):
        raise _bad("kept must be a contiguous int32 tensor [B, Hkv, budget]")
    need = _workspace_bytes("dflash_kv_evict_workspace_bytes", device.index, B, Hkv, N, budget)
    ws = _scratch(need, device)
    _lib.check(_lib.lib().dflash_kv_evict(
        k_cache.data_ptr(), v_cache.data_ptr(), _ptr(page_table), kv_len.data_ptr(), mass.data_ptr(), kv_len_out.data_ptr(),
        mass_out.data_ptr(), _ptr(kept), _ptr(ws), need, B, Hkv, D, N, page_tokens, max_pages, num_pages, mass.shape[2], budget,
        recent, sinks, _DT[k_cache.dtype], _raw_stream(device.index)))
    return kv_len_out


def gated_delta_into(q, k, v, g, beta, state, n_per_seq, y, state_out, tape=None, mask=None) -> None:
    """Allocation-free form of gated_delta_kernel_with_tape: every buffer is supplied by the
    caller (contiguous, on the current device, dtypes as documented there).  state_out may be
    the same tensor as state."""
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    mask_t, mdt = _mask_arg(mask)
    _lib.check(_lib.lib().dflash_gated_delta_tape(
        _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(mask_t), _ptr(n_per_seq),
        _ptr(y), _ptr(state_out), _ptr(tape), B, T, Hk, Hv, Dk, Dv, int(g.dim() == 4), _DT[q.dtype], mdt,
        _stream()))


def batched_sdpa_turbo_kv(queries, k_enc, v_enc, n_cold: int, scale: float, k_hot=None, v_hot=None, out=None) -> Optional[torch.Tensor]:
    """Block-verify attention over KV held in the TurboQuant 3-bit format with a hot window: k_enc = (packed, signs,
    norm, rnorm) and v_enc = (packed, norm) as returned by turbo_encode for the cold history [B,Hkv,n_cold,D]; k_hot,
    v_hot [B,Hkv,n_hot,D] in the attention dtype are the newest tokens (the verify block among them).  With a cold
    history of whole 128-key tiles the library attends in the codec's rotated domain without decoding a key or value
    to global memory; otherwise it expands the cold history into its workspace and attends over the copy
    (dflash_verify_sdpa with DFLASH_KV_TURBO3)."""
    _need_cuda(queries, k_enc[0], v_enc[0])
    B, Hq, T, D = queries.shape
    dt = queries.dtype
    Hkv = k_enc[2].shape[1]
    if T != 16 or dt not in (torch.bfloat16, torch.float16) or D not in (128, 256) or Hq % Hkv != 0:
        return None
    q = queries.contiguous()
    if out is None:
        out = torch.empty_like(q)
    n_hot = 0 if k_hot is None else k_hot.shape[2]
    n_keys = n_cold + n_hot
    L = _lib.lib()
    ws = _workspace(q.device, L.dflash_verify_sdpa_turbo_workspace_bytes(B, Hq, Hkv, D, n_cold, n_hot))
    kp, ks, kn, kr = (t.contiguous() for t in k_enc)
    vp, vn = (t.contiguous() for t in v_enc)
    kh = None if k_hot is None else k_hot.to(dt).contiguous()
    vh = None if v_hot is None else v_hot.to(dt).contiguous()
    desc = _lib.TurboKV(_ptr(kp), _ptr(ks), _ptr(kn), _ptr(kr), _ptr(vp), _ptr(vn), _ptr(kh), _ptr(vh), n_cold, n_hot)
    try:
        _lib.check(L.dflash_verify_sdpa(_ptr(q), C.cast(C.pointer(desc), C.c_void_p), None, None, None, None, _ptr(out),
                                        _ptr(ws), ws.numel(), B, Hq, Hkv, T, D, n_keys, 0, 0, 0, float(scale), _DT[dt],
                                        _lib.KV_TURBO3, _stream()))
    except _lib.DFlashUnsupported:
        return None
    return out


def rebuild_conv_state(conv_snapshot: Optional[torch.Tensor], qkv: torch.Tensor, steps, keep: int) -> torch.Tensor:
    """RecurrentRollbackCache.rebuildConvState (Sources/DFlash/RecurrentRollbackCache.swift:139-158) on the device:
    concat(conv_snapshot [B,keep,C], qkv [B,T,C])[:, steps : min(steps + keep, keep + T)].  `steps` is an int
    (the reference's accepted_steps) or a device int32 tensor [B] of per-sequence step counts (keep rows each)."""
    _need_cuda(qkv)
    qkv = qkv.contiguous()
    B, T, Cdim = qkv.shape
    row_bytes = Cdim * qkv.element_size()
    snap = None if conv_snapshot is None else conv_snapshot.to(qkv.dtype).contiguous()
    rows = C.c_int32(0)
    out = torch.empty(B, keep, Cdim, dtype=qkv.dtype, device=qkv.device)
    if isinstance(steps, torch.Tensor):
        st = steps.to(torch.int32).contiguous()
        _lib.check(_lib.lib().dflash_rebuild_conv_state(_ptr(snap), _ptr(qkv), _ptr(st), 0, _ptr(out), B, T, keep,
                                                       row_bytes, C.byref(rows), _stream()))
        return out
    # scalar count: the window is [B, rows, C] with rows <= keep, written densely at the front of `out`
    end = min(int(steps) + keep, keep + T)
    n_rows = max(end - int(steps), 0)
    out = torch.empty(B, n_rows, Cdim, dtype=qkv.dtype, device=qkv.device)
    if n_rows:
        _lib.check(_lib.lib().dflash_rebuild_conv_state(_ptr(snap), _ptr(qkv), None, int(steps), _ptr(out), B, T, keep,
                                                       row_bytes, C.byref(rows), _stream()))
    return out


def turbo_encode(x: torch.Tensor, is_key: bool):
    """TurboQuant 3-bit encode of 128-dimension blocks (tests/test_turbo_quant.cpp:69-74 for V,
    :85-94 for K in the reference tree).  x [..., 128*m]; returns packed uint8 [..., m, 48],
    signs uint8 [..., m, 16] or None (V), norm and rnorm (or None) as fp16 bit patterns in int16 tensors."""
    _need_cuda(x)
    if x.shape[-1] % 128 != 0:
        raise _lib.DFlashUnsupported(_lib.ERR_UNSUPPORTED, "last dimension must be a multiple of 128")
    x = x.contiguous()
    lead = tuple(x.shape[:-1]) + (x.shape[-1] // 128,)
    n = x.numel() // 128
    packed = torch.empty(lead + (48,), dtype=torch.uint8, device=x.device)
    norm = torch.empty(lead, dtype=torch.int16, device=x.device)
    signs = torch.empty(lead + (16,), dtype=torch.uint8, device=x.device) if is_key else None
    rnorm = torch.empty(lead, dtype=torch.int16, device=x.device) if is_key else None
    _lib.check(_lib.lib().dflash_turbo_encode(_ptr(x), _ptr(packed), _ptr(signs), _ptr(norm), _ptr(rnorm), n,
                                             int(is_key), _DT[x.dtype], _stream()))
    return packed, signs, norm, rnorm


def turbo_decode(packed, signs, norm, rnorm, dtype=torch.bfloat16) -> torch.Tensor:
    """Inverse of turbo_encode (tests/test_turbo_quant.cpp:74-75 and :96-98): returns [..., 128*m]."""
    _need_cuda(packed, norm)
    is_key = signs is not None
    lead = tuple(norm.shape)
    n = norm.numel()
    out = torch.empty(lead[:-1] + (lead[-1] * 128,), dtype=dtype, device=packed.device)
    _lib.check(_lib.lib().dflash_turbo_decode(_ptr(packed.contiguous()), _ptr(signs), _ptr(norm.contiguous()),
                                             _ptr(rnorm), _ptr(out), n, int(is_key), _DT[dtype], _stream()))
    return out
