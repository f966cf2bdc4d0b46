"""Paged cache of exact keys and values, in 16 or 8 bits, and the attention of new tokens over it.

The reference keeps dense [B,H,N,D] caches that every step concatenates to (ops/attn_rerope.py:19-113) and refuses a
second chunk of a prompt ("Only support prefilling or generation", ops/attn_vq.py:247).  Here a cache is two pools of
pages that sequences of any length share:

    k_pages, v_pages [pages, Hkv, page, D]   q's dtype, or torch.float8_e4m3fn with
    k_exp, v_exp     [pages, Hkv, page]      uint8: value = e4m3 * 2^(byte - 127), one byte per row
    block_table      [S, width] int32        the pages of each sequence, in order; -1 (or any number that is no page)
                                             where there is none
    kv_lens          [S] int32               keys of each sequence, new ones included
    cu_q             [S + 1] int32           the new rows of sequence s are the packed rows cu_q[s] .. cu_q[s + 1]

A step is `paged_write(k, v, ...)` and then `attn_paged(q, ...)` with the same table, `cu_q` and `kv_lens`, whether it
brings one token per sequence, chunks of prompts, or both.  `paged_read` gives the cache back as the plain tensors that
the other operators take.  Lengths and tables are read on the device when the kernels run: a step recorded into a HIP
graph replays on new ones.  Sequences of one call must not write to the same page (they may read the same one).
"""
import math

import torch

from .. import _lib
from ._common import SUFFIX, bhn_strides, last_dim_contiguous, ptr

E4M3 = torch.float8_e4m3fn


def _check_pools(k_pages, v_pages, k_exp, v_exp, dtype):
    """(e4m3, page): whether the pools hold 8 bits, and rows per page."""
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "pages must be [pages, heads, page, D], keys and values alike"
    assert k_pages.dtype == v_pages.dtype, "All tensors must have the same type"
    assert dtype in SUFFIX, "Only support fp16 and bf16"
    assert k_pages.shape[3] in (64, 128), "head dimensions 64 and 128 are supported"
    page = k_pages.shape[2]
    assert 16 <= page <= 4096 and page & (page - 1) == 0, "the page size must be a power of two, 16 to 4096"
    assert k_pages.stride(3) == 1 and v_pages.stride(3) == 1, "pages need a contiguous last dimension"
    if k_pages.dtype == E4M3:
        assert k_exp is not None and v_exp is not None, "8-bit pages need k_exp and v_exp"
        for e in (k_exp, v_exp):
            assert e.shape == k_pages.shape[:3] and e.dtype == torch.uint8 and e.stride(2) == 1
        return 1, page
    assert k_exp is None and v_exp is None, "exponents belong to 8-bit pages"
    assert k_pages.dtype == dtype, "All tensors must have the same type"
    return 0, page


def _check_seqs(block_table, kv_lens, cu_q=None):
    assert block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.shape[1] >= 1
    assert block_table.shape[1] == 1 or block_table.stride(1) == 1, "block_table needs contiguous rows"
    S = block_table.shape[0]
    assert kv_lens.shape == (S,) and kv_lens.dtype == torch.int32 and kv_lens.is_contiguous()
    if cu_q is not None:
        assert cu_q.shape == (S + 1,) and cu_q.dtype == torch.int32 and cu_q.is_contiguous()
    return S, block_table.shape[1]


def _check_devices(*tensors):
    _lib.require_gpu(*tensors)
    assert len({t.device for t in tensors if t is not None}) == 1, "All tensors must be on the same device"


def _exp_strides(e):
    return (0, 0) if e is None else (e.stride(0), e.stride(1))


def paged_write(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None):
    """Store the new tokens' rows k, v [T,Hkv,D] in their places, in place: packed row cu_q[s] + t goes to position
    kv_lens[s] - n + t of sequence s (n = cu_q[s + 1] - cu_q[s]).  With 8-bit pages every row is divided by the smallest
    power of two that brings it into e4m3's +-448 and rounded to the nearest; NaN stays NaN, infinities and magnitudes
    beyond 1.875 * 2^15 (fp16) or 1.875 * 2^127 (bf16) are stored as that.  Rows behind the last sequence, before
    position 0, behind the table's last page or on a page that is not there are skipped."""
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype, "k and v must be [T,H,D] of one type"
    e4m3, page = _check_pools(k_pages, v_pages, k_exp, v_exp, k.dtype)
    T, H, D = k.shape
    assert k_pages.shape[1] == H and k_pages.shape[3] == D, "k, v and the pages must have the same heads"
    S, width = _check_seqs(block_table, kv_lens, cu_q)
    _check_devices(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp)
    if T == 0 or S == 0:
        return
    lib = _lib.load()
    k, v = last_dim_contiguous(k, v)
    strides = _lib.strides_array(k.stride(0), k.stride(1), v.stride(0), v.stride(1), *bhn_strides(k_pages),
                                 *bhn_strides(v_pages), *_exp_strides(k_exp), *_exp_strides(v_exp),
                                 block_table.stride(0))
    with torch.cuda.device(k.device):
        rc = getattr(lib, "vqa_paged_write_" + SUFFIX[k.dtype])(
            ptr(k), ptr(v), ptr(k_pages), ptr(v_pages), ptr(k_exp), ptr(v_exp), ptr(block_table), ptr(cu_q),
            ptr(kv_lens), T, S, H, D, page, k_pages.shape[0], width, e4m3, strides, _lib.current_stream(k.device))
    _lib.check(rc)


def paged_read(k_pages, v_pages, block_table, kv_lens, n, *, k_exp=None, v_exp=None, dtype=None):
    """(k, v) [S,Hkv,n,D]: the first n rows of every sequence as plain tensors, zeros from kv_lens[s] on and on pages that
    are not there.  `dtype`: the element type of the result (8-bit pages: required; else the pages' own)."""
    dtype = k_pages.dtype if dtype is None else dtype
    e4m3, page = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    S, width = _check_seqs(block_table, kv_lens)
    assert n >= 0, "the number of rows must not be negative"
    _check_devices(k_pages, v_pages, block_table, kv_lens, k_exp, v_exp)
    P, H, _, D = k_pages.shape
    k = torch.empty((S, H, n, D), dtype=dtype, device=k_pages.device)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    lib = _lib.load()
    strides = _lib.strides_array(*bhn_strides(k_pages), *bhn_strides(v_pages), *_exp_strides(k_exp),
                                 *_exp_strides(v_exp), block_table.stride(0), *bhn_strides(k), *bhn_strides(v))
    with torch.cuda.device(k.device):
        rc = getattr(lib, "vqa_paged_read_" + SUFFIX[dtype])(
            ptr(k_pages), ptr(v_pages), ptr(k_exp), ptr(v_exp), ptr(block_table), ptr(kv_lens), ptr(k), ptr(v), S, H, n,
            D, page, P, width, e4m3, strides, _lib.current_stream(k.device))
    _lib.check(rc)
    return k, v


def attn_paged(q, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None, softmax_scale=None,
               causal=True, window=None, return_lse=False, max_q_len=None, out=None):
    """Attention of the new tokens q [T,Hq,D] over their sequences' cached keys and values (which already hold theirs).

    Row t of sequence s stands at position i = kv_lens[s] - n + t and sees the keys j <= i, with `window` those with
    i - j <= window (the strict rule of `triton_fused_local_attn`); causal=False: every key of its sequence.  Hq is a
    multiple of the pages' heads; query head h reads key head h // (Hq // Hkv).  Returns out [T,Hq,D] (q's dtype) and, with
    return_lse, the base-2 log-sum-exp [T,Hq] fp32: a state `merge_state_in_place` can combine.  A row that sees no key
    gets 0 and -inf; rows behind the last sequence are left as they are (`out`: the buffer to write to).
    `max_q_len`: the most new tokens any sequence has, where the caller knows it; it steers the choice of kernels only."""
    assert q.dim() == 3, "q must be [T,H,D]"
    e4m3, page = _check_pools(k_pages, v_pages, k_exp, v_exp, q.dtype)
    T, Hq, D = q.shape
    P, Hkv = k_pages.shape[:2]
    assert k_pages.shape[3] == D, "q and the pages must have the same head dimension"
    assert Hkv >= 1 and Hq >= 1 and Hq % Hkv == 0, "the query heads must be a multiple of the key heads"
    S, width = _check_seqs(block_table, kv_lens, cu_q)
    assert window is None or (causal and window >= 0), "a window needs causal attention and a length of at least 0"
    softmax_scale = softmax_scale or 1.0 / math.sqrt(D)
    assert softmax_scale > 0, "the softmax scale must be positive"
    assert out is None or (out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1)
    _check_devices(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp, out)
    (q,) = last_dim_contiguous(q)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if T == 0 or S == 0:
        return (out, lse) if return_lse else out
    lib = _lib.load()
    max_q = T if max_q_len is None else max(0, min(int(max_q_len), T))
    ws_bytes = lib.vqa_paged_attn_workspace_bytes(T, S, Hq, Hkv, D, max_q)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    strides = _lib.strides_array(q.stride(0), q.stride(1), *bhn_strides(k_pages), *bhn_strides(v_pages),
                                 *_exp_strides(k_exp), *_exp_strides(v_exp), block_table.stride(0), out.stride(0),
                                 out.stride(1))
    with torch.cuda.device(q.device):
        rc = getattr(lib, "vqa_paged_attn_" + SUFFIX[q.dtype])(
            ptr(q), ptr(k_pages), ptr(v_pages), ptr(k_exp), ptr(v_exp), ptr(block_table), ptr(cu_q), ptr(kv_lens),
            ptr(out), ptr(lse), ptr(ws), ws_bytes, T, S, Hq, Hkv, D, page, P, width, e4m3, strides, 1 if causal else 0,
            -1 if window is None else min(int(window), (1 << 31) - 1), max_q, softmax_scale,
            _lib.current_stream(q.device))
    _lib.check(rc)
    return (out, lse) if return_lse else out
