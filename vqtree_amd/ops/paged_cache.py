"""Paged cache of exact keys and values, in 16 or 8 bits, and the attention of new tokens over it.

The reference keeps dense [B,H,N,D] caches that every step concatenates to (ops/attn_rerope.py:19-113) and refuses a
second chunk of a prompt ("Only support prefilling or generation", ops/attn_vq.py:247).  Here a cache is two pools of
pages that sequences of any length share:

    k_pages, v_pages [pages, Hkv, page, D]   q's dtype, or torch.float8_e4m3fn with
    k_exp, v_exp     [pages, Hkv, page]      uint8: value = e4m3 * 2^(byte - 127), one byte per row (0 counts as 1)
    block_table      [S, width] int32        the pages of each sequence, in order; -1 (or any number that is no page)
                                             where there is none
    kv_lens          [S] int32               keys of each sequence, new ones included
    cu_q             [S + 1] int32           the new rows of sequence s are the packed rows cu_q[s] .. cu_q[s + 1]

A step is `paged_write(k, v, ...)` and then `attn_paged(q, ...)` with the same table, `cu_q` and `kv_lens`, whether it
brings one token per sequence, chunks of prompts, or both.  `paged_read` gives the cache back as the plain tensors that
the other operators take.  Lengths and tables are read on the device when the kernels run: a step recorded into a HIP
graph replays on new ones.  Sequences of one call must not write to the same page (they may read the same one), nor
one sequence to a page that its table names twice.
"""
import math
import operator

import torch

from .. import _lib
from ._common import SUFFIX, last_dim_contiguous

E4M3 = torch.float8_e4m3fn


# A generation step is a few microseconds of GPU work, so the host side counts.  What follows from shapes, strides, types and
# options alone -- the checks, the strides array, the workspace's size -- is worked out once for each combination of them and
# kept (_PLANS); a call then looks that up, checks the devices, and hands over the addresses.  A key holds plain values only:
# a number that comes as a tensor would be found again by its identity, whatever has become of its value.
_PLANS = {}
_MOST_PLANS = 4096


def _remember(key, plan):
    if len(_PLANS) >= _MOST_PLANS:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


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


def _check_devices(dev, *tensors):
    """every tensor is on GPU `dev` (an index; -1: the CPU)"""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _lib.require_gpu(t, *tensors)
            raise AssertionError("All tensors must be on the same device")
    if dev < 0:
        _lib.require_gpu(*tensors)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _sig(x):
    return None if x is None else (x.shape, x.stride(), x.dtype)


def _launch(fn, dev, *args):
    """Calls an entry point on the current stream of device `dev`."""
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _lib.raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc)


def _entry(name, dtype):
    return getattr(_lib.load(), name + SUFFIX[dtype])


def paged_write(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None):
    """Store the new tokens' rows k, v [T,Hkv,D] in their places, in place: packed row cu_q[s] + t goes to position
    kv_lens[s] - n + t of sequence s (n = cu_q[s + 1] - cu_q[s]).  With 8-bit pages every row is divided by the smallest
    power of two that brings it into e4m3's +-448 and rounded to the nearest; NaN stays NaN, infinities and magnitudes
    beyond 1.875 * 2^15 (fp16) or 1.875 * 2^127 (bf16) are stored as that.  Rows behind the last sequence, before
    position 0, behind the table's last page or on a page that is not there are skipped."""
    key = ("w", k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, k_pages.shape, k_pages.stride(), k_pages.dtype,
           v_pages.shape, v_pages.stride(), v_pages.dtype, block_table.shape, block_table.stride(), block_table.dtype,
           cu_q.shape, cu_q.stride(), cu_q.dtype, kv_lens.shape, kv_lens.stride(), kv_lens.dtype, _sig(k_exp), _sig(v_exp))
    plan = _PLANS.get(key) or _remember(key, _plan_write(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp))
    dev = k.get_device()
    _check_devices(dev, k, v, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp)
    fn, tail = plan
    if tail is None:  # a last dimension with gaps, or nothing to do
        if k.numel() and cu_q.numel() > 1:
            paged_write(*last_dim_contiguous(k, v), k_pages, v_pages, block_table, cu_q, kv_lens, k_exp=k_exp, v_exp=v_exp)
        return
    _launch(fn, dev, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp), _ptr(v_exp),
            block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), *tail)


def _plan_write(k, v, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp):
    shape, dtype = k.shape, k.dtype
    assert len(shape) == 3 and shape == v.shape and dtype == v.dtype, "k and v must be [T,H,D] of one type"
    T, H, D = shape
    e4m3, pages, strides, exp_strides = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    assert pages[1] == H and pages[3] == D, "k, v and the pages must have the same heads"
    S, width, table_stride = _check_seqs(block_table, kv_lens, cu_q)
    if T == 0 or S == 0 or k.stride(2) != 1 or v.stride(2) != 1:
        return None, None
    strides = _lib.strides_array(*k.stride()[:2], *v.stride()[:2], *strides, *exp_strides, table_stride)
    return _entry("vqa_paged_write_", dtype), (T, S, H, D, pages[2], pages[0], width, e4m3, strides)


def paged_read(k_pages, v_pages, block_table, kv_lens, n, *, k_exp=None, v_exp=None, dtype=None):
    """(k, v) [S,Hkv,n,D]: the first n rows of every sequence as plain tensors, zeros from kv_lens[s] on and on pages that
    are not there.  `dtype`: the element type of the result (8-bit pages: required; else the pages' own)."""
    n = operator.index(n)
    key = ("r", k_pages.shape, k_pages.stride(), k_pages.dtype, v_pages.shape, v_pages.stride(), v_pages.dtype,
           block_table.shape, block_table.stride(), block_table.dtype, kv_lens.shape, kv_lens.stride(), kv_lens.dtype,
           _sig(k_exp), _sig(v_exp), n, dtype)
    plan = _PLANS.get(key) or _remember(key, _plan_read(k_pages, v_pages, block_table, kv_lens, n, k_exp, v_exp, dtype))
    dev = k_pages.get_device()
    _check_devices(dev, k_pages, v_pages, block_table, kv_lens, k_exp, v_exp)
    fn, shape, dtype, tail = plan
    k, v = k_pages.new_empty(shape, dtype=dtype), k_pages.new_empty(shape, dtype=dtype)
    if tail is not None:
        _launch(fn, dev, k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp), _ptr(v_exp), block_table.data_ptr(),
                kv_lens.data_ptr(), k.data_ptr(), v.data_ptr(), *tail)
    return k, v


def _plan_read(k_pages, v_pages, block_table, kv_lens, n, k_exp, v_exp, dtype):
    dtype = k_pages.dtype if dtype is None else dtype
    e4m3, pages, strides, exp_strides = _check_pools(k_pages, v_pages, k_exp, v_exp, dtype)
    S, width, table_stride = _check_seqs(block_table, kv_lens)
    assert n >= 0, "the number of rows must not be negative"
    P, H, page, D = pages
    if S == 0 or n == 0 or H == 0:
        return None, (S, H, n, D), dtype, None
    out = (H * n * D, n * D, D)
    strides = _lib.strides_array(*strides, *exp_strides, table_stride, *out, *out)
    return _entry("vqa_paged_read_", dtype), (S, H, n, D), dtype, (S, H, n, D, page, P, width, e4m3, strides)


def attn_paged(q, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None, softmax_scale=None,
               causal=True, window=None, return_lse=False, max_q_len=None, out=None):
    """Attention of the new tokens q [T,Hq,D] over their sequences' cached keys and values (which already hold theirs).

    Row t of sequence s stands at position i = kv_lens[s] - n + t and sees the keys j <= i, with `window` those with
    i - j <= window (the strict rule of `triton_fused_local_attn`); causal=False: every key of its sequence.  Hq is a
    multiple of the pages' heads; query head h reads key head h // (Hq // Hkv).  Returns out [T,Hq,D] (q's dtype) and, with
    return_lse, the base-2 log-sum-exp [T,Hq] fp32: a state `merge_state_in_place` can combine.  A row that sees no key
    gets 0 and -inf; rows behind the last sequence are left as they are (`out`: the buffer to write to).
    `max_q_len`: the most new tokens any sequence has, where the caller knows it; it steers the choice of kernels only.
    For the number of keys that choice goes by what block_table has room for."""
    causal = bool(causal)
    if softmax_scale is not None:
        softmax_scale = float(softmax_scale)
    if window is not None:
        window = int(window)
    if max_q_len is not None:
        max_q_len = int(max_q_len)
    key = ("a", q.shape, q.stride(), q.dtype, k_pages.shape, k_pages.stride(), k_pages.dtype, v_pages.shape,
           v_pages.stride(), v_pages.dtype, block_table.shape, block_table.stride(), block_table.dtype, cu_q.shape,
           cu_q.stride(), cu_q.dtype, kv_lens.shape, kv_lens.stride(), kv_lens.dtype, _sig(k_exp), _sig(v_exp), _sig(out),
           softmax_scale, causal, window, max_q_len)
    plan = _PLANS.get(key) or _remember(key, _plan_attn(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp,
                                                        softmax_scale, causal, window, max_q_len, out))
    dev = q.get_device()
    _check_devices(dev, q, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp, out)
    fn, ws_bytes, tail = plan
    if tail is None and q.numel() and kv_lens.numel():  # a last dimension with gaps
        return attn_paged(q.contiguous(), k_pages, v_pages, block_table, cu_q, kv_lens, k_exp=k_exp, v_exp=v_exp,
                          softmax_scale=softmax_scale, causal=causal, window=window, return_lse=return_lse,
                          max_q_len=max_q_len, out=out)
    if out is None:
        out = q.new_empty(q.shape)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    if tail is not None:
        ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        _launch(fn, dev, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_exp), _ptr(v_exp),
                block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(ws), ws_bytes,
                *tail)
    return (out, lse) if return_lse else out


def _plan_attn(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_exp, v_exp, softmax_scale, causal, window, max_q_len, out):
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
    if T == 0 or S == 0 or q.stride(2) != 1:
        return None, 0, None
    lib = _lib.load()
    max_q = T if max_q_len is None else max(0, min(max_q_len, T))
    causal = 1 if causal else 0
    window = -1 if window is None else min(window, (1 << 31) - 1)
    ws_bytes = lib.vqa_paged_attn_workspace_bytes(T, S, Hq, Hkv, D, page, width, e4m3, causal, window, max_q)
    out_strides = (Hq * D, D) if out is None else out.stride()[:2]
    strides = _lib.strides_array(*q.stride()[:2], *strides, *exp_strides, table_stride, *out_strides)
    return _entry("vqa_paged_attn_", dtype), ws_bytes, (T, S, Hq, Hkv, D, page, P, width, e4m3, strides, causal, window,
                                                        max_q, softmax_scale)
