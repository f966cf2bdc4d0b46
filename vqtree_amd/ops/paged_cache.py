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
import functools
import math

import torch

from .. import _lib
from ._common import SUFFIX, last_dim_contiguous

E4M3 = torch.float8_e4m3fn


# A generation step is a few microseconds of GPU work, so the host side counts: attributes are read once, the device is
# switched only where it has to be.
def _check_pools(k_pages, v_pages, k_exp, v_exp, dtype):
    """(e4m3, page shape, strides of the pools, strides of the exponents)"""
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    assert len(shape) == 4 and shape == v_pages.shape, "pages must be [pages, heads, page, D], keys and values alike"
    pages_dtype = k_pages.dtype
    assert pages_dtype == v_pages.dtype, "All tensors must have the same type"
    assert dtype in SUFFIX, "Only support fp16 and bf16"
    page, D = shape[2], shape[3]
    assert D == 128 or D == 64, "head dimensions 64 and 128 are supported"
    assert 16 <= page <= 4096 and page & (page - 1) == 0, "the page size must be a power of two, 16 to 4096"
    assert ks[3] == 1 and vs[3] == 1, "pages need a contiguous last dimension"
    strides = (*ks[:3], *vs[:3])
    if pages_dtype == E4M3:
        assert k_exp is not None and v_exp is not None, "8-bit pages need k_exp and v_exp"
        es, fs = k_exp.stride(), v_exp.stride()
        assert k_exp.shape == v_exp.shape == shape[:3] and k_exp.dtype == v_exp.dtype == torch.uint8
        assert es[2] == 1 and fs[2] == 1, "exponents need a contiguous last dimension"
        return 1, shape, strides, (*es[:2], *fs[:2])
    assert k_exp is None and v_exp is None, "exponents belong to 8-bit pages"
    assert pages_dtype == dtype, "All tensors must have the same type"
    return 0, shape, strides, (0, 0, 0, 0)


def _check_seqs(block_table, kv_lens, cu_q=None):
    """(S, width, stride of a table row)"""
    shape, stride = block_table.shape, block_table.stride()
    assert len(shape) == 2 and block_table.dtype == torch.int32, "block_table must be [S, width] int32"
    S, width = shape
    assert width >= 1 and (width == 1 or stride[1] == 1), "block_table needs contiguous rows"
    assert kv_lens.shape == (S,) and kv_lens.dtype == torch.int32 and kv_lens.is_contiguous()
    if cu_q is not None:
        assert cu_q.shape == (S + 1,) and cu_q.dtype == torch.int32 and cu_q.is_contiguous()
    return S, width, stride[0]


def _check_devices(*tensors):
    """index of the device all of them are on"""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _lib.require_gpu(t, tensors[0])
            raise AssertionError("All tensors must be on the same device")
    _lib.require_gpu(tensors[0])
    return dev


def _ptr(x):
    return None if x is None else x.data_ptr()


def _launch(name, dtype, dev, *args):
    """Calls the entry point of the element type on the current stream of device `dev`."""
    fn = getattr(_lib.load(), name + SUFFIX[dtype])
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _lib.raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc)


@functools.lru_cache(maxsize=1024)
def _attn_workspace_bytes(*sizes):
    return _lib.load().vqa_paged_attn_workspace_bytes(*sizes)


def paged_write(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None):
    """Store the new tokens' rows k, v [T,Hkv,D] in their places, in place: packed row cu_q[s] + t goes to position
    kv_lens[s] - n + t of sequence s (n = cu_q[s + 1] - cu_q[s]).  With 8-bit pages every row is divided by the smallest
    power of two that brings it into e4m3's +-448 and rounded to the nearest; NaN stays NaN, infinities and magnitudes
    beyond 1.875 * 2^15 (fp16) or 1.875 * 2^127 (bf16) are stored as that.  Rows behind the last sequence, before
    position 0, behind the table's last page or on a page that is not there are skipped."""
    shape, dtype = k.shape, k.dtype
    assert len(shape) == 3 and shape == v.shape and dtype == v.dtype, "k and v must be [T,H,D] of one type"
    T, H, D = shape
    e4m3, pages, strides, exp_strides = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    assert pages[1] == H and pages[3] == D, "k, v and the pages must have the same heads"
    S, width, table_stride = _check_seqs(block_table, kv_lens, cu_q)
    dev = _check_devices(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp)
    if T == 0 or S == 0:
        return
    k, v = last_dim_contiguous(k, v)
    strides = _lib.strides_array(*k.stride()[:2], *v.stride()[:2], *strides, *exp_strides, table_stride)
    _launch("vqa_paged_write_", dtype, dev, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp),
            _ptr(v_exp), block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), T, S, H, D, pages[2], pages[0], width,
            e4m3, strides)


def paged_read(k_pages, v_pages, block_table, kv_lens, n, *, k_exp=None, v_exp=None, dtype=None):
    """(k, v) [S,Hkv,n,D]: the first n rows of every sequence as plain tensors, zeros from kv_lens[s] on and on pages that
    are not there.  `dtype`: the element type of the result (8-bit pages: required; else the pages' own)."""
    dtype = k_pages.dtype if dtype is None else dtype
    e4m3, pages, strides, exp_strides = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    S, width, table_stride = _check_seqs(block_table, kv_lens)
    assert n >= 0, "the number of rows must not be negative"
    dev = _check_devices(k_pages, v_pages, block_table, kv_lens, k_exp, v_exp)
    P, H, page, D = pages
    k = torch.empty((S, H, n, D), dtype=dtype, device=k_pages.device)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    strides = _lib.strides_array(*strides, *exp_strides, table_stride, *k.stride()[:3], *v.stride()[:3])
    _launch("vqa_paged_read_", dtype, dev, k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp), _ptr(v_exp),
            block_table.data_ptr(), kv_lens.data_ptr(), k.data_ptr(), v.data_ptr(), S, H, n, D, page, P, width, e4m3, strides)
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
    shape, dtype = q.shape, q.dtype
    assert len(shape) == 3, "q must be [T,H,D]"
    T, Hq, D = shape
    e4m3, pages, strides, exp_strides = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    P, Hkv, page, pages_dim = pages
    assert pages_dim == D, "q and the pages must have the same head dimension"
    assert Hkv >= 1 and Hq >= 1 and Hq % Hkv == 0, "the query heads must be a multiple of the key heads"
    S, width, table_stride = _check_seqs(block_table, kv_lens, cu_q)
    assert window is None or (causal and window >= 0), "a window needs causal attention and a length of at least 0"
    softmax_scale = softmax_scale or 1.0 / math.sqrt(D)
    assert softmax_scale > 0, "the softmax scale must be positive"
    assert out is None or (out.shape == shape and out.dtype == dtype and out.stride(2) == 1)
    dev = _check_devices(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp, out)
    (q,) = last_dim_contiguous(q)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if T == 0 or S == 0:
        return (out, lse) if return_lse else out
    max_q = T if max_q_len is None else max(0, min(int(max_q_len), T))
    causal = 1 if causal else 0
    window = -1 if window is None else min(int(window), (1 << 31) - 1)
    ws_bytes = _attn_workspace_bytes(T, S, Hq, Hkv, D, page, width, e4m3, causal, window, max_q)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    strides = _lib.strides_array(*q.stride()[:2], *strides, *exp_strides, table_stride, *out.stride()[:2])
    _launch("vqa_paged_attn_", dtype, dev, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp), _ptr(v_exp),
            block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(ws), ws_bytes, T, S,
            Hq, Hkv, D, page, P, width, e4m3, strides, causal, window, max_q, softmax_scale)
    return (out, lse) if return_lse else out
